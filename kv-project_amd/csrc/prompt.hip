// Attention over whole prompts: packed sequences of any lengths, grouped heads, causal with the last
// query at the last key (a chunk of a prompt behind its past) or over all keys.
//
// A workgroup takes 128 rows of one KV head: (token, query head) pairs, token major, so that the query
// heads of a group share the keys and values that are staged in LDS, 64 tokens at a time.  Each of its
// four wavefronts holds 32 rows as the columns of the matrix products: S^T = K Q^T, the softmax in base
// 2 with one running reference and sum per column (two lanes hold a column; one swap joins them), and
// O^T += V^T P^T.  The accumulator layout of S^T is the operand layout of P^T once V^T takes its tokens in
// the same order, so probabilities never leave their lanes: V^T comes from LDS by transposing reads.
// Probabilities are rounded to the inputs' type (half a step of the output's type); the sums, the
// references and the accumulators are float32.  fp16 has no room below 2^-24: there the reference weighs 2^7, so that
// weights lose at most 2^-32 of it (200000 keys of 2^-26 each, 0.3% of the sum, were zeros without).
//
// Where the rows are too few to fill the chip, a tile of rows is cut along its keys into parts, each
// with its own sums, and prompt_merge_kernel joins them in order.
//
// What bounds it: the matrix cores and the power they draw.  One causal prompt of 16384 tokens, 32 query heads over 8
// KV heads of 128, bf16: 1913-2085 us by card (1.06-1.15 PFLOP/s; a library product of the largest size reaches 1.36),
// matrix cores busy 62%, vector unit 55% of the cycles, at 1.7 GHz of 2.4; no LDS conflicts; keys and values come
// from memory 4.5 times, otherwise from the caches.  With head_dim 64 a score costs half the products and the same
// exponential, so the vector unit leads (68%; matrix cores 42%): four sequences of 512 to 1531 tokens behind up to 9000,
// 235-253 us (0.81-0.87 PFLOP/s; 250-283 traced over 30 passes).  24 sequences of 1 to 2901 tokens, fp16, head_dim 128:
// 172-188 us (0.73-0.80 PFLOP/s; 179-214 traced): 71 iterations for each of 512 places, 133 us at the long prompt's rate,
// and the starts and ends of five tiles.  20 tokens: 7 us, a launch and the round trips of one tile.
// Measured and not kept: 64 rows a wavefront (half the LDS reads, but accumulators move between the register files:
// 2040-2680 us); sums by a product with ones at head_dim 64 (235 -> 258 us); other wave priorities (3-5% slower);
// workgroups that stay for several tiles and fetch the next one's first keys during the last steps (24 sequences of 256
// tokens 61 -> 54 us, but 3% slower over 273 shapes and 9% at head_dim 64, for its registers).
#include <algorithm>
#include <cfloat>
#include <cmath>
#include <type_traits>

#include "mfma_common.hpp"

namespace kvq {
namespace {

constexpr int kThreads = 256, kTileRows = 128, kTileKeys = 64, kItemWords = 8, kSlots = 512, kMinPart = 8;

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
typedef __attribute__((address_space(3))) void lds_void;

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

// In each group of 16 lanes, lane 4 k + j names 4 values of row k; lane i receives column i of the four rows.
__device__ __forceinline__ u32x2 read_tr(const uint16_t* p) {
  return __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(p)));
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

struct PromptArgs {
  const uint16_t *q, *k, *v;
  int64_t q_st, q_sh, k_st, k_sh, v_st, v_sh;
  const int* items;                           // {first row, tokens, first key, keys, visible to the first token, step, part or -1}
  int H, rep;
  float scale;                                // |scaling| * log2(e)
  uint32_t sign;                              // of scaling, for both halves of a word of q
  uint16_t* out;                              // (rows, Hq, D)
  float* part;                                // (parts, H): 128 x D sums, then 128 x {reference, sum}
};

// Iteration j takes a tile of 64 tokens through the softmax, beside matrix products that do not depend on it:
// O += V(j-1) P(j-1); then S(j+1) = K(j+1) Q, alone, while the other wavefront of the SIMD is in its
// softmax.  The order is written down step by step (a step is one operand from LDS, one product and a
// share of the softmax) and fenced.  K(j+2) and V(j) go from memory to LDS during the iteration (two buffers each, one
// barrier an iteration); the number of tiles is rounded up to an odd one, so that buffers and registers of even
// and odd tiles have fixed places.
template <int D, bool BF16>
__global__ __launch_bounds__(kThreads, 2) void prompt_kernel(PromptArgs a) {
  constexpr int kRow = D / 8, kPer = kTileKeys * kRow / kThreads;   // 16-byte pieces of a row, of a thread
  constexpr int kBuf = kTileKeys * D;                               // elements of a buffer
  constexpr uint32_t kInf = BF16 ? 0x7f80u : 0x7c00u;
  constexpr int kTiles = 5;                   // tiles that some row sees in part: 128 tokens, two ends, one of padding
  __shared__ __align__(16) uint16_t k_even[kBuf], k_odd[kBuf], v_even[kBuf], v_odd[kBuf];
  __shared__ int flag[kTiles];
  const int* it = a.items + kItemWords * (blockIdx.x / a.H);
  const int h = blockIdx.x % a.H;
  const int row0 = it[0], toks = it[1], key0 = it[2], keys = it[3], vis0 = it[4], vis_step = it[5];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, col = lane & 31, g = lane >> 5;

  const int row = wave * 32 + col, tok = row / a.rep, hq = row % a.rep;
  const bool live = tok < toks;
  const int sees = vis0 + vis_step * tok, visible = !live ? 0 : sees < keys ? sees : keys;
  // every lane reads a row, dead ones the first: a select of the result becomes a branch around each load, one round trip
  // after the other (24 sequences of 256 tokens 60 us, 65 so)
  u32x4 q[D / 16];
  const uint32_t mask = live ? ~0u : 0u;
  const uint16_t* qp = a.q + (row0 + static_cast<int64_t>(live ? tok : 0)) * a.q_st + (static_cast<int64_t>(h) * a.rep + hq) * a.q_sh + 8 * g;
  each<0, D / 16>([&](auto i) { q[i.value] = *reinterpret_cast<const u32x4*>(qp + 16 * i.value); });
  f32x16 o[D / 32], s[2][2];                  // s, p: of even and odd tiles
  float m = -INFINITY, l = 0.0f, grow = 1.0f; // the exponents' reference, this lane's part of the sum, what o is to be scaled by
  u32x4 p[2][4];
  each<0, D / 32>([&](auto c) { each<0, 16>([&](auto e) { o[c.value][e.value] = 0.0f; }); });

  // A thread's pieces of a tile: 16 bytes, the x-th of LDS, x = tid + i kThreads: row x / kRow, place x % kRow.
  // A piece c of row r lies at place c ^ k_swz(r) or c ^ v_swz(r) of its row, so that 16 lanes of a read of K (16
  // rows, one piece) and 32 of a read of V (4 rows, two pieces in two places) meet 256 different bytes of the banks.
  auto k_swz = [](int r) { return D == 128 ? r & 15 : r >> 1 & 7; };
  auto v_swz = [](int r) { return D == 128 ? (r & 3) << 2 : (r >> 1 & 1) << 2; };
  const int xr = tid / kRow, xc = tid % kRow;
  constexpr int kStep = kThreads / kRow;      // rows from one piece to the next: a multiple of kRow
  const uint16_t* kb = a.k + static_cast<int64_t>(key0) * a.k_st + h * a.k_sh;
  const uint16_t* vb = a.v + static_cast<int64_t>(key0) * a.v_st + h * a.v_sh;
  const int k_at = (xr * static_cast<int>(a.k_st) + (xc ^ k_swz(xr)) * 8) * 2;
  const int v_at = (xr * static_cast<int>(a.v_st) + (xc ^ v_swz(xr)) * 8) * 2;
  const int wave0 = __builtin_amdgcn_readfirstlane(wave) * 512;     // elements
  // Straight to LDS, 16 bytes a lane, written down here so that it can run beside the transposing reads (the compiler
  // has those wait for every load to LDS).  m0 is set by the compiler, which so knows of it; end() waits.
  auto fetch = [&](uint16_t* to, const uint16_t* base, int64_t st, int at, int j) KVQ_INLINE {
    // rows behind the last one read as zeros: the buffer ends with the last row
    const int64_t left = keys - static_cast<int64_t>(j) * kTileKeys;
    const int64_t bytes = left > 0 ? ((left - 1) * st + D) * 2 : 0;
    const uint64_t from = reinterpret_cast<uint64_t>(base + (left > 0 ? static_cast<int64_t>(j) * kTileKeys * st : 0));
    const u32x4 rsrc = {static_cast<uint32_t>(from), static_cast<uint32_t>(from >> 32) & 0xffffu,
                        static_cast<uint32_t>(bytes < 0x7fffffff ? bytes : 0x7fffffff), 0x00020000u};
    const uint32_t lds = static_cast<uint32_t>(reinterpret_cast<uintptr_t>((lds_void*)(to + wave0)));
#pragma unroll
    for (int i = 0; i < kPer; ++i)
      asm volatile("s_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds"
                   :
                   : "{m0}"(lds + i * kThreads * 16), "v"(at + i * kStep * static_cast<int>(st) * 2), "s"(rsrc)
                   : "memory");
  };
  const int tiles = ((keys + kTileKeys - 1) / kTileKeys) | 1;
  int open = vis0 < keys ? vis0 : keys;       // tiles that every row sees whole
  open = open < 0 ? 0 : open / kTileKeys;

  const int k_x = g ^ k_swz(col);             // piece 2 i + g of row 32 x + col lies at piece (2 i) ^ k_x
  auto read_k = [&](auto par, int t) KVQ_INLINE {        // operand t of K: channels 16 (t / 2) .., rows 32 (t % 2) ..
    return *reinterpret_cast<const u32x4*>((decltype(par)::value ? k_odd : k_even) + col * D + ((2 * (t / 2)) ^ k_x) * 8 + 32 * (t % 2) * D);
  };
  // 16 tokens a product; this lane's: 16 y + 4 g + e and 16 y + 8 + 4 g + e.  The transposing read of row
  // 16 y + 8 e + 4 g + tr: channels 32 c + 16 (lane / 16 % 2) + 4 (lane % 4) .. lie at piece (4 c) ^ v_x
  const int tr = (lane & 15) >> 2, v_x = ((lane >> 4 & 1) * 2 + (lane >> 1 & 1)) ^ v_swz(4 * g + tr);
  auto read_v = [&](auto par, int t) KVQ_INLINE {        // operand t of V^T: tokens 16 y .., channels 32 c ..
    const int y = t / (D / 32), c = t % (D / 32);
    const uint16_t* base = (decltype(par)::value ? v_odd : v_even) + (4 * g + tr) * D + (lane & 1) * 4 + ((4 * c) ^ v_x) * 8 + 16 * y * D;
    const u32x2 u = read_tr(base), w = read_tr(base + 8 * D);
    return u32x4{u[0], u[1], w[0], w[1]};
  };
  // the softmax of tile j in 18 shares: 0 and 1 find the reference, 2 + i the weights 2 i, 2 i + 1.
  // register 16 x + 4 b + e of lane half g: token 32 x + 8 b + 4 g + e
  constexpr float kLift = BF16 ? 0.0f : 7.0f; // log2 of the reference's weight
  float top, safe, sum;
  auto share = [&](auto par, bool masked, int j, auto which) KVQ_INLINE {
    constexpr int i = decltype(which)::value;
    auto& t = s[decltype(par)::value];
    if constexpr (i < 2) {
      if (masked) {
        const int lim = visible - j * kTileKeys - 4 * g;
        each<0, 16>([&](auto e) KVQ_INLINE { t[i][e.value] = 32 * i + 8 * (e.value / 4) + e.value % 4 < lim ? t[i][e.value] : -INFINITY; });
      }
      float x = i == 0 ? t[0][0] : fmaxf(top, t[1][0]);
      each<1, 16>([&](auto e) KVQ_INLINE { x = fmaxf(x, t[i][e.value]); });
      top = x;
      if constexpr (i == 1) {
        // the reference moves only when a score passes it by 2^8: weights up to 256 (fp16: 2^15) cost no accuracy, and the
        // accumulators are hardly ever scaled
        x = xmax32(x) * a.scale;
        x = x > m + 8.0f ? x : m;
        safe = x == -INFINITY ? 0.0f : x;
        grow = __builtin_amdgcn_exp2f(m - safe);
        safe -= kLift;
        m = x;
        sum = 0.0f;
      }
    } else {
      constexpr int k = 2 * (i - 2);
      const float x = __builtin_amdgcn_exp2f(__builtin_fmaf(t[k / 16][k % 16], a.scale, -safe));
      const float z = __builtin_amdgcn_exp2f(__builtin_fmaf(t[k / 16][k % 16 + 1], a.scale, -safe));
      sum += x;
      sum += z;
      uint32_t w = pack2<BF16>(x, z);
      asm volatile("" : "+v"(w));             // here, not behind the branch of the rescaling
      p[decltype(par)::value][k / 8][k % 8 / 2] = w;
      if constexpr (i == 17) {
        l = l * grow + sum;
        asm volatile("" : "+v"(l));
      }
    }
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
  // o += V(j-1) P(j-1) (if `with`) beside the softmax of tile j
  auto values = [&](auto par, bool masked, auto with, int j) KVQ_INLINE {
    constexpr bool kWith = decltype(with)::value;
    constexpr std::integral_constant<int, 1 - decltype(par)::value> other{};
    u32x4 w[3];
    if constexpr (kWith) {
      w[0] = read_v(other, 0);
      w[1] = read_v(other, 1);
    }
    each<0, kV>([&](auto t) KVQ_INLINE {
      if constexpr (kWith) {
        if constexpr (t.value + 2 < kV) w[(t.value + 2) % 3] = read_v(other, t.value + 2);
        add_v(other, t, w[t.value % 3]);
      }
      each<t.value * 18 / kV, (t.value + 1) * 18 / kV>([&](auto i) KVQ_INLINE { share(par, masked, j, i); });
      __builtin_amdgcn_sched_barrier(0);
    });
  };
  auto products = [&](auto par) KVQ_INLINE {  // S = K Q of the tiles of the other parity
    constexpr int next = 1 - decltype(par)::value;
    constexpr std::integral_constant<int, next> other{};
    u32x4 w[4];
    each<0, 16>([&](auto e) KVQ_INLINE { s[next][0][e.value] = s[next][1][e.value] = 0.0f; });
    each<0, 3>([&](auto t) KVQ_INLINE { w[t.value] = read_k(other, t.value); });
    each<0, kK>([&](auto t) KVQ_INLINE {
      if constexpr (t.value + 3 < kK) w[(t.value + 3) % 4] = read_k(other, t.value + 3);
      s[next][t.value % 2] = mfma32<BF16>(w[t.value % 4], q[t.value / 2], s[next][t.value % 2]);
      __builtin_amdgcn_sched_barrier(0);
    });
  };
  auto rescale = [&]() KVQ_INLINE {
    if (__builtin_amdgcn_ballot_w64(grow != 1.0f)) each<0, D / 32>([&](auto c) KVQ_INLINE { o[c.value] *= grow; });
  };
  // A value that is hidden from some row may be an infinity or a NaN: in LDS it becomes a zero, and the rows that
  // do see it have it at the end.  A thread looks at the pieces that it fetched itself.
  auto watch = [&](uint16_t* to, int j) KVQ_INLINE {
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      u32x4* at = reinterpret_cast<u32x4*>(to + (tid + i * kThreads) * 8);
      u32x4 w = *at;
      bool bad = false;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const bool b0 = (w[e] & kInf) == kInf, b1 = (w[e] >> 16 & kInf) == kInf;
        bad |= b0 || b1;
        w[e] = (b0 ? 0u : w[e] & 0xffffu) | (b1 ? 0u : w[e] & 0xffff0000u);
      }
      if (bad) {
        *at = w;
        flag[j - open] = 1;
      }
    }
  };
  auto begin = [&](auto par, int j) KVQ_INLINE {
    fetch(decltype(par)::value ? k_odd : k_even, kb, a.k_st, k_at, j + 2);
    fetch(decltype(par)::value ? v_odd : v_even, vb, a.v_st, v_at, j);
    __builtin_amdgcn_sched_barrier(0);
  };
  auto end = [&](auto par, int j) KVQ_INLINE {
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");                // this wavefront's pieces are in LDS
    if (j >= open) watch(decltype(par)::value ? v_odd : v_even, j);
    __syncthreads();
  };
  auto step = [&](auto par, int j) KVQ_INLINE {
    begin(par, j);
    __builtin_amdgcn_s_setprio(1);            // the softmax goes before the other wavefront's products
    values(par, j >= open, yes, j);
    __builtin_amdgcn_s_setprio(0);
    products(par);
    rescale();
    end(par, j);
  };
  if (keys > 0) {
    if (tid < kTiles) flag[tid] = 0;
    __syncthreads();
    fetch(k_even, kb, a.k_st, k_at, 0);
    fetch(v_even, vb, a.v_st, v_at, 0);
    if (tiles > 1) fetch(k_odd, kb, a.k_st, k_at, 1);
    each<0, D / 16>([&](auto i) KVQ_INLINE { q[i.value] = (q[i.value] ^ a.sign) & mask; });
    end(even, 0);
    products(odd);
    if (tiles > 1) {
      __syncthreads();                        // K(2) takes the place of K(0)
      fetch(k_even, kb, a.k_st, k_at, 2);
      __builtin_amdgcn_sched_barrier(0);
    }
    values(even, open == 0, no, 0);
    if (tiles > 1) {
      products(even);
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      __syncthreads();
    }
    for (int j = 1; j < tiles; j += 2) {
      step(odd, j);
      step(even, j + 1);
    }
    each<0, kV>([&](auto t) KVQ_INLINE { add_v(even, t, read_v(even, t.value)); });
    // A visible value that is infinite or NaN is its channel's result, however small its weight has become (zero times it would
    // be a NaN).  In tiles that every row sees it has made the sum infinite or NaN: they are looked through, each lane 8 channels
    // of every (64 / kRow)-th token (bits e, 8 + e, 16 + e: an infinity, a negative one, a NaN in channel e).  In the others
    // it was left out of the sum.
    l = xsum32(l);
    float all = 0.0f;
    each<0, D / 32>([&](auto c) KVQ_INLINE { each<0, 16>([&](auto e) KVQ_INLINE { all += o[c.value][e.value]; }); });
    if (__builtin_amdgcn_ballot_w64(live && l == l && !finite(all))) {
      uint32_t found = 0;
#pragma unroll 8
      for (int r = lane / kRow; r < open * kTileKeys; r += 64 / kRow) {
        const u32x4 w = *reinterpret_cast<const u32x4*>(vb + r * a.v_st + lane % kRow * 8);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const uint32_t x = w[e / 2] >> (16 * (e % 2)) & 0xffffu;
          if ((x & kInf) == kInf) found |= 1u << (e + ((x & 0x7fffu) != kInf ? 16 : x >> 15 ? 8 : 0));
        }
      }
#pragma unroll
      for (int i = kRow; i < 64; i *= 2) found |= __shfl_xor(found, i);
      each<0, D / 8>([&](auto i) KVQ_INLINE {
        const uint32_t f = __shfl(found, i.value) >> (4 * g);
        each<0, 4>([&](auto e) KVQ_INLINE {
          const bool up = f >> e.value & 1, down = f >> (8 + e.value) & 1, nan = f >> (16 + e.value) & 1;
          auto& x = o[i.value / 4];
          constexpr int at = i.value % 4 * 4 + e.value;
          x[at] = nan || (up && down) ? NAN : up ? INFINITY : down ? -INFINITY : x[at];
        });
      });
    }
    for (int j = open; j < tiles; ++j)
      if (flag[j - open])
        for (int r = j * kTileKeys; r < j * kTileKeys + kTileKeys && r < keys; ++r)
          each<0, D / 32>([&](auto c) KVQ_INLINE {
            each<0, 16>([&](auto e) KVQ_INLINE {
              const uint16_t x = vb[r * a.v_st + 32 * c.value + 8 * (e.value / 4) + 4 * g + e.value % 4];
              if (r < visible && (x & kInf) == kInf) o[c.value][e.value] += BF16 ? bf16_to_f32(x) : f16_to_f32(x);
            });
          });
  }

  if (!live) return;
  const int piece = it[6];
  if (piece >= 0) {
    float* part = a.part + (static_cast<int64_t>(piece) * a.H + h) * (kTileRows * (D + 2));
    each<0, D / 32>([&](auto c) KVQ_INLINE {
      each<0, 4>([&](auto e) KVQ_INLINE {
        const auto& x = o[c.value];
        *reinterpret_cast<float4*>(part + row * D + 32 * c.value + 8 * e.value + 4 * g) =
            make_float4(x[4 * e.value], x[4 * e.value + 1], x[4 * e.value + 2], x[4 * e.value + 3]);
      });
    });
    if (g == 0) *reinterpret_cast<float2*>(part + kTileRows * D + 2 * row) = make_float2(m, l);
    return;
  }
  const float inv = visible > 0 ? 1.0f / l : 0.0f;                  // a row without a visible key: zeros
  uint16_t* out = a.out + ((row0 + static_cast<int64_t>(tok)) * a.H * a.rep + h * a.rep + hq) * D + 4 * g;
  each<0, D / 32>([&](auto c) KVQ_INLINE {
    each<0, 4>([&](auto e) KVQ_INLINE {
      const auto& x = o[c.value];
      *reinterpret_cast<uint2*>(out + 32 * c.value + 8 * e.value) =
          make_uint2(pack2<BF16>(x[4 * e.value] * inv, x[4 * e.value + 1] * inv), pack2<BF16>(x[4 * e.value + 2] * inv, x[4 * e.value + 3] * inv));
    });
  });
}

// One wavefront per row of a tile that was cut, the references of 64 parts at a time.  merges[i] = {first part, parts, first row, tokens}
template <int D, bool BF16>
__global__ __launch_bounds__(kThreads) void prompt_merge_kernel(PromptArgs a, const int* __restrict__ merges) {
  const int* w = merges + 4 * (blockIdx.x / a.H);
  const int h = blockIdx.x % a.H, lane = threadIdx.x & 63, row = blockIdx.y * (kThreads / 64) + (threadIdx.x >> 6);
  const int tok = row / a.rep, parts = w[1];
  if (tok >= w[3]) return;
  constexpr int64_t kPart = kTileRows * (D + 2);
  const int64_t stride = a.H * kPart;
  const float* part = a.part + (static_cast<int64_t>(w[0]) * a.H + h) * kPart;
  float top = -INFINITY, l = 0.0f, o[D / 64] = {};
  for (int i0 = 0; i0 < parts; i0 += 64) {
    const int i = i0 + lane;
    const float2 st = i < parts ? *reinterpret_cast<const float2*>(part + i * stride + kTileRows * D + 2 * row) : make_float2(-INFINITY, 0.0f);
    const float m = fmaxf(top, wave_max(st.x)), safe = m == -INFINITY ? 0.0f : m;
    const float old = __builtin_amdgcn_exp2f(top - safe), f = __builtin_amdgcn_exp2f(st.x - safe);
    l = l * old + wave_sum(f * st.y);
#pragma unroll
    for (int e = 0; e < D / 64; ++e) o[e] = weigh(old, o[e]);
    const int most = parts - i0 < 64 ? parts - i0 : 64;
    for (int k = 0; k < most; ++k) {
      const float fk = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(f), k));
      const float* x = part + (i0 + k) * stride + row * D + lane * (D / 64);
#pragma unroll
      for (int e = 0; e < D / 64; ++e) o[e] += weigh(fk, x[e]);
    }
    top = m;
  }
  const float inv = 1.0f / l;                 // a tile that was cut has a visible key for every row
  uint16_t* out = a.out + ((w[2] + static_cast<int64_t>(tok)) * a.H * a.rep + h * a.rep + row % a.rep) * D + lane * (D / 64);
#pragma unroll
  for (int e = 0; e < D / 64; ++e) out[e] = BF16 ? f32_to_bf16(o[e] * inv) : f32_to_f16(o[e] * inv);
}

struct Item {
  int32_t w[kItemWords];
};

}  // namespace
}  // namespace kvq

using namespace kvq;

extern "C" int kvq_prompt_plan(const int64_t* lens_q, const int64_t* lens_k, int64_t n, int64_t rep, int64_t H, int causal, int32_t* words,
                               int64_t words_cap, int64_t* info) {
  KVQ_REQUIRE(info && n >= 0 && (n == 0 || (lens_q && lens_k)), "kvq_prompt_plan: null pointer");
  KVQ_REQUIRE(rep >= 1 && rep <= kTileRows && H >= 1, "kvq_prompt_plan: bad head counts");
  const int64_t per_tile = kTileRows / rep;   // tokens of a tile of rows
  int64_t rows = 0, keys_all = 0, tiles = 0, longest = 0;
  auto keys_of = [&](int64_t i, int64_t t) {  // keys that the tile from token t of sequence i sees
    if (!causal) return lens_k[i];
    const int64_t end = t + per_tile < lens_q[i] ? t + per_tile : lens_q[i], k = lens_k[i] - lens_q[i] + end;
    return k < 0 ? INT64_C(0) : k;
  };
  auto steps_of = [&](int64_t i, int64_t t) { return (keys_of(i, t) + kTileKeys - 1) / kTileKeys; };
  for (int64_t i = 0; i < n; ++i) {
    KVQ_REQUIRE(lens_q[i] >= 0 && lens_k[i] >= 0, "kvq_prompt_plan: lengths must not be negative");
    rows += lens_q[i];
    keys_all += lens_k[i];
    KVQ_REQUIRE(rows < INT64_C(1) << 31 && keys_all < INT64_C(1) << 31, "kvq_prompt_plan: too many rows");
    for (int64_t t = 0; t < lens_q[i]; t += per_tile, ++tiles) longest = steps_of(i, t) > longest ? steps_of(i, t) : longest;
  }
  // Where the tiles of rows do not fill kSlots places (two on each of 256 CUs), they are cut into the shortest parts that
  // fit: 8 key tiles at least, which pay for the part's sums (64 KB).  Parts beyond the places start a second round, which
  // costs more than uneven ones: 8 sequences of 1024 tokens, 8 heads of 128, 512 tiles whole 36 us, 768 parts of an even
  // share at most 53; 24 of 16 tokens behind 32768, 384 parts 605, 576 of them 723.  Batches whose tiles fill the places
  // stay whole, however uneven: 64 tokens behind 60000 beside twelve prompts of 256 (32 query heads over 8) wait for
  // tiles of 939 steps, 33 of them an even share.
  int64_t most = kMinPart, high = longest > kMinPart ? longest : kMinPart;
  if (tiles * H > kSlots) most = high;
  while (most < high) {
    const int64_t mid = (most + high) / 2;
    int64_t count = 0;
    for (int64_t i = 0; i < n; ++i)
      for (int64_t t = 0; t < lens_q[i]; t += per_tile) count += steps_of(i, t) > mid ? (steps_of(i, t) + mid - 1) / mid : 1;
    if (count * H <= kSlots) high = mid;
    else most = mid + 1;
  }
  int64_t items = 0, merges = 0, parts = 0;
  Item* out = reinterpret_cast<Item*>(words);
  for (int pass = 0; pass < 2; ++pass) {
    int64_t row = 0, key = 0, item = 0, part = 0, merge = 0;
    for (int64_t i = 0; i < n; ++i) {
      for (int64_t t = 0; t < lens_q[i]; t += per_tile) {
        const int64_t toks = lens_q[i] - t < per_tile ? lens_q[i] - t : per_tile, keys = keys_of(i, t);
        const int64_t vis0 = causal ? lens_k[i] - lens_q[i] + t + 1 : keys, steps = steps_of(i, t);
        const int64_t cut = (steps + most - 1) / most, count = cut > 1 ? cut : 1;
        if (pass == 1 && count > 1) {
          int32_t* w = words + kItemWords * items + 4 * merge;
          w[0] = static_cast<int32_t>(part);
          w[1] = static_cast<int32_t>(count);
          w[2] = static_cast<int32_t>(row + t);
          w[3] = static_cast<int32_t>(toks);
        }
        for (int64_t c = 0; c < count; ++c, ++item) {
          const int64_t first = steps * c / count * kTileKeys, last = steps * (c + 1) / count * kTileKeys;
          if (pass == 1)
            out[item] = {{static_cast<int32_t>(row + t), static_cast<int32_t>(toks), static_cast<int32_t>(key + first),
                          static_cast<int32_t>((last < keys ? last : keys) - first), static_cast<int32_t>(vis0 - first), causal ? 1 : 0,
                          count > 1 ? static_cast<int32_t>(part + c) : -1, 0}};
        }
        if (count > 1) {
          part += count;
          ++merge;
        }
      }
      row += lens_q[i];
      key += lens_k[i];
    }
    items = item;
    merges = merge;
    parts = part;
    info[0] = items;
    info[1] = merges;
    info[2] = parts;
    if (!words || words_cap < kItemWords * items + 4 * merges) return KVQ_OK;
  }
  // the longest first: the last workgroups to end are short ones
  std::sort(out, out + items, [](const Item& x, const Item& y) {
    return x.w[3] != y.w[3] ? x.w[3] > y.w[3] : x.w[2] != y.w[2] ? x.w[2] < y.w[2] : x.w[0] < y.w[0];
  });
  return KVQ_OK;
}

extern "C" int64_t kvq_prompt_workspace(int64_t parts, int64_t H, int64_t D) {
  return parts < 0 || H < 1 || (D != 64 && D != 128) ? -1 : parts * H * kTileRows * (D + 2);
}

extern "C" int kvq_prompt_attention(const void* q, int64_t q_st, int64_t q_sh, const void* k, int64_t k_st, int64_t k_sh, const void* v,
                                    int64_t v_st, int64_t v_sh, int dtype, int64_t Hq, int64_t H, int64_t D, float scaling,
                                    const int32_t* words, int64_t items, int64_t merges, int64_t parts, void* out, float* workspace,
                                    int64_t workspace_floats, void* stream) {
  KVQ_REQUIRE(D == 64 || D == 128, "kvq_prompt_attention: head_dim must be 64 or 128 (got %lld)", static_cast<long long>(D));
  KVQ_REQUIRE(dtype == KVQ_F16 || dtype == KVQ_BF16, "kvq_prompt_attention: rows must be fp16 or bf16");
  KVQ_REQUIRE(H > 0 && Hq > 0 && Hq % H == 0 && Hq / H <= kTileRows && items >= 0 && merges >= 0 && parts >= 0, "kvq_prompt_attention: bad sizes");
  if (items == 0) return KVQ_OK;
  KVQ_REQUIRE(q && k && v && words && out, "kvq_prompt_attention: null pointer");
  KVQ_REQUIRE((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v) |
               reinterpret_cast<uintptr_t>(out) | reinterpret_cast<uintptr_t>(workspace)) % 16 == 0 && (q_st | q_sh | k_st | k_sh | v_st | v_sh) % 8 == 0,
              "kvq_prompt_attention: rows and strides must be multiples of 16 bytes");
  KVQ_REQUIRE(items * H <= kMaxGrid && merges * H <= kMaxGrid, "kvq_prompt_attention: too many rows");
  KVQ_REQUIRE(k_st >= 0 && v_st >= 0 && k_st < (1 << 24) && v_st < (1 << 24), "kvq_prompt_attention: row strides must be below 2^24 elements");
  KVQ_REQUIRE(parts == 0 || (workspace && workspace_floats >= kvq_prompt_workspace(parts, H, D)),
              "kvq_prompt_attention: workspace of %lld floats, %lld needed", static_cast<long long>(workspace_floats),
              static_cast<long long>(kvq_prompt_workspace(parts, H, D)));
  // a scaling of nothing would make a NaN of a hidden score's -inf: the smallest one, which makes zeros of the others
  const float scale = std::fabs(scaling) * 1.44269504088896341f;
  const PromptArgs a{static_cast<const uint16_t*>(q), static_cast<const uint16_t*>(k), static_cast<const uint16_t*>(v),
                     q_st, q_sh, k_st, k_sh, v_st, v_sh, words, static_cast<int>(H), static_cast<int>(Hq / H),
                     scale < FLT_MIN ? FLT_MIN : scale, std::signbit(scaling) ? 0x80008000u : 0u,
                     static_cast<uint16_t*>(out), workspace};
  const dim3 grid(static_cast<uint32_t>(items * H)), joins(static_cast<uint32_t>(merges * H), kTileRows * 64 / kThreads);
  hipStream_t s = static_cast<hipStream_t>(stream);
  auto run = [&](auto d, auto t) {
    hipLaunchKernelGGL((prompt_kernel<decltype(d)::value, decltype(t)::value>), grid, dim3(kThreads), 0, s, a);
    if (merges)
      hipLaunchKernelGGL((prompt_merge_kernel<decltype(d)::value, decltype(t)::value>), joins, dim3(kThreads), 0, s, a, words + kItemWords * items);
  };
  auto by_type = [&](auto d) {
    if (dtype == KVQ_BF16) run(d, std::true_type{});
    else run(d, std::false_type{});
  };
  if (D == 64) by_type(std::integral_constant<int, 64>{});
  else by_type(std::integral_constant<int, 128>{});
  KVQ_LAUNCH_CHECK("kvq_prompt_attention");
  return KVQ_OK;
}
