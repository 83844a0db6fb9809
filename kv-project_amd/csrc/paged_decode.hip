// Attention of a few query tokens per sequence over the paged 8-bit cache (layouts: pages.hpp).
//
// Rows of a KV head: (query token, query head) pairs, 16 to a workgroup, the columns of the matrix
// products.  A unit is 64 tokens; a wavefront computes its scores S = K q (rows tokens, columns query
// rows), the running maximum and sum of the softmax in base 2, and O += V^T P, all in registers:
//   S tile s of a unit takes token 16 (m >> 2) + 4 s + (m & 3) as its row m, so lane group g = lane / 16 ends
//   up with the scores of tokens 16 g .. 16 g + 15, which is the K-index order that V^T (channel major in the
//   page) is read in with 16 bytes a lane.  No value crosses lanes but the maximum.
// The key scale multiplies the scores, the value scale the probabilities; the codes themselves turn to
// 16-bit numbers exactly.  Probabilities times scale keep 16 bits as a pair of bfloat16 (the range of a
// scale is float32's), so they round at 2^-17.
//
// Workgroups take the units of one split item, their wavefronts in turn, and join in LDS.  A sequence of
// several items is joined in the items' order: by the workgroup that comes last, where tickets are given, or
// by paged_merge_kernel, which spreads long joins over the chip.
//
// What bounds it: long caches, the codes' way from memory: 16 sequences of 32768 tokens, 8 KV heads of 128, 186-201 us
// for 1.07 GB (5.4-5.8 TB/s, 88-94% of the 6.1 TB/s of a read-only stream; the matrix cores are busy 10% of the time, the
// vector unit, which widens the codes, 33%), and 4.7 us of joins.  One sequence of 4096 tokens, 128 workgroups: 8.8 us,
// the round trips of one unit: description, page number, codes, join.  Registers for two workgroups a CU instead
// of three were no faster.
#include <type_traits>

#include "mfma_common.hpp"
#include "pages.hpp"

namespace kvq {
namespace {

constexpr int kThreads = 256, kWaves = 4, kRows = 16;

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef float f32x2 __attribute__((ext_vector_type(2)));

template <bool BF16>
__device__ __forceinline__ f32x4 mfma16(u32x4 a, u32x4 b, f32x4 c) {
  if constexpr (BF16) return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  else return __builtin_amdgcn_mfma_f32_16x16x32_f16(as_half8(a), as_half8(b), c, 0, 0, 0);
}

__device__ __forceinline__ uint32_t pack_bf16(float a, float b) {
  const f32x2 v = {a, b};
  return __builtin_bit_cast(uint32_t, __builtin_convertvector(v, bf16x2));
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
    a = pack_bf16(static_cast<float>(static_cast<int8_t>(s)), static_cast<float>(static_cast<int8_t>(s >> 8)));
    b = pack_bf16(static_cast<float>(static_cast<int8_t>(s >> 16)), static_cast<float>(static_cast<int8_t>(s >> 24)));
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

struct DecodeArgs {
  const uint16_t* q;
  int64_t q_st, q_sh;
  const int* step;
  int n;                                      // sequences of the step
  const int* table;
  int64_t max_blocks;
  int H, rep;                                 // KV heads, query heads per KV head
  int pieces;                                 // of 16 rows, of the widest run
  float scale;                                // scaling * log2(e)
  const uint8_t *kc, *vc;
  const float* sc;
  const uint16_t *ko, *vo;
  uint16_t* out;                              // (rows, Hq, D)
  float* part;                                // (part_rows, H): D sums; behind them {max, sum} each
  int64_t part_rows;                          // rows of all split items
  bool all;                                   // rows are no tokens of their slots: they see all tokens before
  int* tickets;                               // (slots, H, kApart) zeros, or none: joins by a launch of its own
};
constexpr int kApart = 32;                    // a cache line for each ticket: 208 workgroups 10.7 us, 12.2 with them side by side

template <int D, bool BF16>
struct Wave {                                 // one wavefront's running softmax: column lane % 16
  f32x4 o[D / 16];                            // channels 16 c + 4 g + i
  float m, l;                                 // base-2 maximum (of all groups), this lane's part of the sum
};

// Values that workgroups on other dies read in this launch: stores and loads at the level that the dies share, past
// their own caches (a release fence writes a whole cache back: 50 us where 768 workgroups have one each)
__device__ __forceinline__ void put_shared(float* p, float x) { __hip_atomic_store(p, x, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }
template <bool SHARED>
__device__ __forceinline__ float get(const float* p) {
  if constexpr (SHARED) return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  else return *p;
}

// N rows joined by one wavefront: the maxima, the sums, its channels of the weighted sums.  LONG: of many items, 32 on
// their way at once
template <int D, bool SHARED, int N, bool LONG = false>
struct Join {
  float top[N], l[N], o[N][D / 64];
  __device__ __forceinline__ Join() {
#pragma unroll
    for (int n = 0; n < N; ++n) {
      top[n] = -INFINITY;
      l[n] = 0.0f;
#pragma unroll
      for (int e = 0; e < D / 64; ++e) o[n][e] = 0.0f;
    }
  }
  // DEEP items of every row on their way at once; behind the last: it again, unused
  template <int DEEP>
  struct Items {
    float x[N][DEEP][D / 64];
    __device__ __forceinline__ void load(const float* const (&p)[N], int64_t stride, int k0, int most) {
#pragma unroll
      for (int n = 0; n < N; ++n)
#pragma unroll
        for (int k = 0; k < DEEP; ++k)
#pragma unroll
          for (int e = 0; e < D / 64; ++e) x[n][k][e] = get<SHARED>(p[n] + (k0 + k < most ? k0 + k : most - 1) * stride * D + e);
    }
    __device__ __forceinline__ void add_to(Join& j, int k0, int most, const float (&f)[N]) const {
#pragma unroll
      for (int n = 0; n < N; ++n)
#pragma unroll
        for (int k = 0; k < DEEP; ++k) {
          const float fk = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(f[n]), k0 + k < most ? k0 + k : 0));
#pragma unroll
          for (int e = 0; e < D / 64; ++e) j.o[n][e] += k0 + k < most ? weigh(fk, x[n][k][e]) : 0.0f;
        }
    }
  };
  template <int DEEP>
  __device__ __forceinline__ void some(const float* const (&p)[N], int64_t stride, int k0, int most, const float (&f)[N]) {
    Items<DEEP> x;
    x.load(p, stride, k0, most);
    x.add_to(*this, k0, most, f);
  }
  // rows R of a run's split items from .. to - 1, 64 maxima at a time
  __device__ __forceinline__ void add(const DecodeArgs& a, const StepRun& run, const int (&R)[N], int h, int from, int to) {
    const int lane = threadIdx.x & 63;
    const int64_t stride = static_cast<int64_t>(a.rep) * run.tokens * a.H;
    const float* stat = a.part + a.part_rows * a.H * D;
    for (int i0 = from; i0 < to; i0 += 64) {
      const int i = i0 + lane, most = to - i0 < 64 ? to - i0 : 64;
      float2 st[N];
      const float* p[N];
#pragma unroll
      for (int n = 0; n < N; ++n) {
        const int64_t first = (static_cast<int64_t>(a.rep) * run.base + R[n]) * a.H + h;
        p[n] = a.part + (first + i0 * stride) * D + lane * (D / 64);
        st[n] = make_float2(-INFINITY, 0.0f);
        if (i < to) st[n] = make_float2(get<SHARED>(stat + 2 * (first + i * stride)), get<SHARED>(stat + 2 * (first + i * stride) + 1));
      }
      Items<8> early;                         // on their way with the maxima
      early.load(p, stride, 0, most);
      float f[N];
#pragma unroll
      for (int n = 0; n < N; ++n) {
        const float m = fmaxf(top[n], wave_max(st[n].x)), safe = m == -INFINITY ? 0.0f : m;
        const float old = __builtin_amdgcn_exp2f(top[n] - safe);
        f[n] = __builtin_amdgcn_exp2f(st[n].x - safe);
        l[n] = l[n] * old + wave_sum(f[n] * st[n].y);
#pragma unroll
        for (int e = 0; e < D / 64; ++e) o[n][e] = weigh(old, o[n][e]);
        top[n] = m;
      }
      early.add_to(*this, 0, most, f);
      int k0 = 8;
      if constexpr (LONG)
        for (; k0 + 32 <= most; k0 += 32) some<32>(p, stride, k0, most, f);
      for (; k0 < most; k0 += 8) some<8>(p, stride, k0, most, f);
    }
  }
  template <bool BF16>
  __device__ __forceinline__ void put(int n, uint16_t* out) const {
    const float inv = 1.0f / l[n];
#pragma unroll
    for (int e = 0; e < D / 64; ++e) out[(threadIdx.x & 63) * (D / 64) + e] = BF16 ? f32_to_bf16(o[n][e] * inv) : f32_to_f16(o[n][e] * inv);
  }
};

// Rows wave, wave + kWaves, .. of a sequence (N of them at most) out of its split items, within the launch that made them
template <int D, bool BF16, int N>
__device__ __forceinline__ void join_rows(const DecodeArgs& a, const StepRun& run, int wave, int rows, int h) {
  int R[N];
#pragma unroll
  for (int n = 0; n < N; ++n) R[n] = wave + n * kWaves < rows ? wave + n * kWaves : rows - 1;
  Join<D, true, N> j;
  j.add(a, run, R, h, 0, run.items);
#pragma unroll
  for (int n = 0; n < N; ++n)
    if (wave + n * kWaves < rows)
      j.template put<BF16>(n, a.out + ((static_cast<int64_t>(run.row0) + R[n] / a.rep) * a.H * a.rep + h * a.rep + R[n] % a.rep) * D);
}

// Scores t (16 tokens of this lane, masked ones -inf) -> probabilities in t, o and l brought to the new maximum
template <int D, bool BF16>
__device__ __forceinline__ void soft(Wave<D, BF16>& w, float (&t)[16]) {
  float m = t[0];
#pragma unroll
  for (int i = 1; i < 16; ++i) m = fmaxf(m, t[i]);
  m = fmaxf(w.m, xmax32(xmax16(m)));
  const float safe = m == -INFINITY ? 0.0f : m;
  const float a = __builtin_amdgcn_exp2f(w.m - safe);
  float sum = 0.0f;
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    t[i] = __builtin_amdgcn_exp2f(t[i] - safe);
    sum += t[i];
  }
  w.l = w.l * a + sum;
  if (__builtin_amdgcn_ballot_w64(a != 1.0f)) {
#pragma unroll
    for (int c = 0; c < D / 16; ++c) w.o[c] *= a;
  }
  w.m = m;
}

__device__ __forceinline__ void split_bf16(const float (&p)[16], int at, u32x4& hi, u32x4& lo) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float a = p[at + 2 * i], b = p[at + 2 * i + 1];
    const uint32_t h = pack_bf16(a, b);
    hi[i] = h;
    lo[i] = pack_bf16(a - __uint_as_float(h << 16), b - __uint_as_float(h & 0xffff0000u));
  }
}
__device__ __forceinline__ void split_f16(const float (&p)[16], int at, u32x4& hi, u32x4& lo) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const _Float16 a = static_cast<_Float16>(p[at + 2 * i]), b = static_cast<_Float16>(p[at + 2 * i + 1]);
    hi[i] = pack_h2(a, b);
    lo[i] = pack_h2(static_cast<_Float16>(p[at + 2 * i] - static_cast<float>(a)), static_cast<_Float16>(p[at + 2 * i + 1] - static_cast<float>(b)));
  }
}

template <int D, int P, int CODE, bool BF16>
__global__ __launch_bounds__(kThreads, 3) void paged_split_kernel(DecodeArgs a) {
  constexpr int kJ = D / 64, kC = D / 16;
  __shared__ float join[kWaves][kRows][D + 4];
  __shared__ float stat[kWaves][kRows][2];
  const int* step = a.step;
  const int per = step[3];
  // pieces of one item and head on one of the 8 dies, next to each other: they read the same pages
  const int group = blockIdx.x / (8 * a.pieces), within = blockIdx.x % (8 * a.pieces);
  const int64_t ih = static_cast<int64_t>(group) * 8 + within % 8;
  const int piece = within / 8, item = static_cast<int>(ih / a.H), h = static_cast<int>(ih % a.H);
  const int* runs = step_runs(step, a.n);
  // no look where a run is one item, or one sequence the only run: that run is read with the header (there is room for
  // 2 n + 1 of them)
  const int near = a.n == 1 ? 0 : item < a.n ? item : a.n;
  StepRun run = step_run(runs, near);
  if (item >= step[2]) return;
  int ri = near;
  if (a.n > 1 && !(step[11] && item == near)) {
    ri = __builtin_amdgcn_readfirstlane(last_not_above(runs + 5, kStepRun, step[8], item));
    run = step_run(runs, ri);
  }
  const int rows = a.rep * run.tokens;
  if (piece * kRows >= rows) return;
  const bool own = run.seq >= 0;              // or a shared front: whole pages that every row sees
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), col = lane & 15, g = lane >> 4;
  const int pos0 = own ? run.pos0 : run.u1 * kUnit, len = own && !a.all ? run.pos0 + run.tokens : pos0, full = len / P * P;
  const int u_full = (full + kUnit - 1) / kUnit;
  const int u0 = run.u0 + (item - run.split0) * per, u1 = u0 + per < run.u1 ? u0 + per : run.u1;

  // the query rows: column col of B, channels 64 j + 16 g + 8 e ..
  const int row = piece * kRows + col, tok = row / a.rep, hq = row % a.rep;
  const bool live = row < rows;
  const int visible = !live ? 0 : a.all ? len : pos0 + tok + 1;
  u32x4 q[2 * kJ];
  {
    const uint16_t* qp = a.q + (run.row0 + (live ? tok : 0)) * a.q_st + (static_cast<int64_t>(h) * a.rep + (live ? hq : 0)) * a.q_sh;
#pragma unroll
    for (int j = 0; j < kJ; ++j)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const uint4 x = *reinterpret_cast<const uint4*>(qp + 64 * j + 16 * g + 8 * e);
        q[2 * j + e] = live ? u32x4{x.x, x.y, x.z, x.w} : u32x4{0, 0, 0, 0};
      }
  }

  Wave<D, BF16> w;
#pragma unroll
  for (int c = 0; c < kC; ++c) w.o[c] = f32x4{0, 0, 0, 0};
  w.m = -INFINITY;
  w.l = 0.0f;

  const int m_tok = 16 * (col >> 2) + (col & 3);                    // + 4 s: the token of S row `col` in tile s
  const int* pages = a.table + run.slot * a.max_blocks;
  const int last = full / P - 1;                                    // last full block
  const int u_end = u1 < u_full ? u1 : u_full;
  // The registers of a unit: keys and its scales are read for the next unit once the scores are there, values once
  // they are added, page numbers a unit further ahead.  With pages of 64 tokens or more a unit lies in one
  // page: its address and scales are scalars, the lanes' offsets constants.
  constexpr bool kOne = P >= kUnit;
  u32x4 kw[4][kJ], vw[kC];
  float2 z;
  int pk, pv;                                 // pages of this lane's key rows and value tokens
  const uint8_t* vp;
  const uint32_t k_off = m_tok * D + 16 * g, v_off = col * P + 16 * g;
  auto ids = [&](int u) {
    if constexpr (kOne) {
      pk = pages[u * kUnit / P];
    } else {
      const int bk = (u * kUnit + m_tok) / P, bv = (u * kUnit + 16 * g) / P;
      pk = pages[bk < last ? bk : last];      // half a unit may lie behind the last page: masked
      pv = pages[bv < last ? bv : last];
    }
  };
  auto keys = [&](int u) {
    const int t0 = u * kUnit;
    const uint8_t* kp;
    if constexpr (kOne) {
      const int64_t at = static_cast<int64_t>(pk) * a.H + h;
      kp = a.kc + at * (P * D) + (t0 & (P - 1)) * D;
      vp = a.vc + at * (P * D) + (t0 & (P - 1));
      z = reinterpret_cast<const float2*>(a.sc)[at];
    } else {
      const int64_t at = static_cast<int64_t>(pv) * a.H + h;
      kp = a.kc + (static_cast<int64_t>(pk) * a.H + h) * (P * D) + (m_tok & (P - 1)) * D + 16 * g;
      vp = a.vc + at * (P * D) + col * P + (16 * g & (P - 1));
      z = reinterpret_cast<const float2*>(a.sc)[at];
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < kJ; ++j) kw[i][j] = *reinterpret_cast<const u32x4*>(kp + (kOne ? k_off + 4 * i * D + 64 * j : 4 * i * D + 64 * j));
  };
  auto values = [&]() {
#pragma unroll
    for (int c = 0; c < kC; ++c) vw[c] = *reinterpret_cast<const u32x4*>(vp + (kOne ? v_off + 16 * c * P : 16 * c * P));
  };
  int u = u0 + wave;
  if (u < u_end) {
    ids(u);
    keys(u);
    values();
    if (u + kWaves < u_end) ids(u + kWaves);
  }
  for (; u < u_end; u += kWaves) {
    const int t0 = u * kUnit;
    const bool more = u + kWaves < u_end;
    float t[16];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      f32x4 acc = {0, 0, 0, 0};
#pragma unroll
      for (int j = 0; j < kJ; ++j) {
        acc = mfma16<BF16>(widen8<CODE, BF16>(kw[i][j][0], kw[i][j][1]), q[2 * j], acc);
        acc = mfma16<BF16>(widen8<CODE, BF16>(kw[i][j][2], kw[i][j][3]), q[2 * j + 1], acc);
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) t[4 * i + e] = acc[e] * (z.x * a.scale);
    }
    const float vz = z.y;
    if (more) {
      keys(u + kWaves);
      if (u + 2 * kWaves < u_end) ids(u + 2 * kWaves);
    }
    const int end = visible < full ? visible : full;
    const bool masked = t0 + kUnit > full || t0 + kUnit > pos0 + 1;
    if (masked) {
#pragma unroll
      for (int i = 0; i < 16; ++i) t[i] = t0 + 16 * g + i < end ? t[i] : -INFINITY;
    }
    soft(w, t);
#pragma unroll
    for (int i = 0; i < 16; ++i) t[i] *= vz;
    if (masked) {                                                   // a NaN scale of a block that no row sees
#pragma unroll
      for (int i = 0; i < 16; ++i) t[i] = t0 + 16 * g + i < end ? t[i] : 0.0f;
    }
    u32x4 hi[2], lo[2];
    split_bf16(t, 0, hi[0], lo[0]);
    split_bf16(t, 8, hi[1], lo[1]);
#pragma unroll
    for (int c = 0; c < kC; ++c) {
      const u32x4 x = widen8<CODE, true>(vw[c][0], vw[c][1]), y = widen8<CODE, true>(vw[c][2], vw[c][3]);
      w.o[c] = mfma16<true>(x, hi[0], w.o[c]);
      w.o[c] = mfma16<true>(y, hi[1], w.o[c]);
      w.o[c] = mfma16<true>(x, lo[0], w.o[c]);
      w.o[c] = mfma16<true>(y, lo[1], w.o[c]);
    }
    if (more) values();
  }

  // Units of the open block.  32-bit offsets from its scalar base and a few loads at a time: their registers must
  // not count for the loop above.
  const int64_t open = ((static_cast<int64_t>(run.slot) * 2 + run.open) * a.H + h) * P * D;
  const uint16_t *ko = a.ko + open, *vo = a.vo + open;
  for (; u < u1; u += kWaves) {
    const int off = (u - u_full) * kUnit, t0 = full + off;
    float t[16];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int r = off + m_tok + 4 * i < P ? off + m_tok + 4 * i : P - 1;   // behind a page of 32 tokens: masked
      f32x4 acc = {0, 0, 0, 0};
#pragma unroll
      for (int j = 0; j < kJ; ++j)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const u32x4 x = *reinterpret_cast<const u32x4*>(ko + static_cast<uint32_t>(r * D + 64 * j + 16 * g + 8 * e));
          acc = mfma16<BF16>(x, q[2 * j + e], acc);
        }
#pragma unroll
      for (int e = 0; e < 4; ++e) t[4 * i + e] = t0 + 16 * g + 4 * i + e < visible ? acc[e] * a.scale : -INFINITY;
      __builtin_amdgcn_sched_barrier(0);
    }
    soft(w, t);
    u32x4 hi[2], lo[2];
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      if constexpr (BF16) split_bf16(t, 8 * e, hi[e], lo[e]);
      else split_f16(t, 8 * e, hi[e], lo[e]);
    }
    // what lies behind the sequence or is hidden from a row may be an infinity or a NaN: it goes in as zero, and
    // the rows that do see such a value have it in that channel, however small its weight: a wavefront has one unit of the open
    // block at most, its last, and the joins keep it
    constexpr uint32_t kInf = BF16 ? 0x7f80u : 0x7c00u;
    const uint32_t at = col * P + (off + 16 * g < P ? off + 16 * g : 0);
    uint32_t worst = 0;
#pragma unroll
    for (int c = 0; c < kC; ++c) {
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        u32x4 v = *reinterpret_cast<const u32x4*>(vo + (at + 16 * c * P + 8 * e));
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const uint32_t b0 = v[i] & kInf, b1 = v[i] >> 16 & kInf;
          worst = b0 > worst ? b0 : worst;
          worst = b1 > worst ? b1 : worst;
          v[i] = (b0 == kInf ? 0u : v[i] & 0xffffu) | (b1 == kInf ? 0u : v[i] & 0xffff0000u);
        }
        w.o[c] = mfma16<BF16>(v, hi[e], w.o[c]);
        w.o[c] = mfma16<BF16>(v, lo[e], w.o[c]);
      }
      __builtin_amdgcn_sched_barrier(0);
    }
    if (__builtin_amdgcn_ballot_w64(worst == kInf)) {
      for (int i = 0; i < kUnit && t0 + i < len; ++i)
#pragma unroll
        for (int c = 0; c < kC; ++c) {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const uint16_t x = vo[static_cast<uint32_t>((16 * c + 4 * g + e) * P + off + i)];
            if ((x & kInf) == kInf && t0 + i < visible) w.o[c][e] += BF16 ? bf16_to_f32(x) : f16_to_f32(x);
          }
          __builtin_amdgcn_sched_barrier(0);
        }
    }
  }

  w.l = xsum32(xsum16(w.l));
#pragma unroll
  for (int c = 0; c < kC; ++c) *reinterpret_cast<f32x4*>(&join[wave][col][16 * c + 4 * g]) = w.o[c];
  if (g == 0) {
    stat[wave][col][0] = w.m;
    stat[wave][col][1] = w.l;
  }
  __syncthreads();
  const bool single = own && run.items == 1 && run.front == 0;
  constexpr int kPer = kRows * D / kThreads;                        // channels of a row per thread
  const int r = threadIdx.x / (D / kPer), c0 = threadIdx.x % (D / kPer) * kPer;
  float top = stat[0][r][0];
#pragma unroll
  for (int i = 1; i < kWaves; ++i) top = fmaxf(top, stat[i][r][0]);
  const float safe = top == -INFINITY ? 0.0f : top;
  float l = 0.0f, o[kPer] = {};
#pragma unroll
  for (int i = 0; i < kWaves; ++i) {
    const float f = __builtin_amdgcn_exp2f(stat[i][r][0] - safe);
    l += f * stat[i][r][1];
#pragma unroll
    for (int e = 0; e < kPer; ++e) o[e] += weigh(f, join[i][r][c0 + e]);
  }
  const int R = piece * kRows + r;
  const int64_t Hq = static_cast<int64_t>(a.H) * a.rep;
  if (single) {
    if (R >= rows) return;
    const float inv = len ? 1.0f / l : 0.0f;  // rows of a slot without tokens: zeros
    uint16_t* out = a.out + ((static_cast<int64_t>(run.row0) + R / a.rep) * Hq + h * a.rep + R % a.rep) * D + c0;
    uint32_t p[kPer / 2];
#pragma unroll
    for (int e = 0; e < kPer / 2; ++e)
      p[e] = BF16 ? pack_bf16(o[2 * e] * inv, o[2 * e + 1] * inv)
                  : pack_h2(static_cast<_Float16>(o[2 * e] * inv), static_cast<_Float16>(o[2 * e + 1] * inv));
#pragma unroll
    for (int e = 0; e < kPer / 4; ++e) *reinterpret_cast<uint2*>(out + 4 * e) = make_uint2(p[2 * e], p[2 * e + 1]);
    return;
  }
  const int64_t at = (static_cast<int64_t>(a.rep) * (run.base + static_cast<int64_t>(item - run.split0) * run.tokens) + R) * a.H + h;
  float *part = a.part + at * D, *st = a.part + a.part_rows * a.H * D + 2 * at;
  if (!a.tickets) {
    if (R >= rows) return;
#pragma unroll
    for (int e = 0; e < kPer / 4; ++e)
      *reinterpret_cast<float4*>(part + c0 + 4 * e) = make_float4(o[4 * e], o[4 * e + 1], o[4 * e + 2], o[4 * e + 3]);
    if (c0 == 0) *reinterpret_cast<float2*>(st) = make_float2(top, l);
    return;
  }
  if (R < rows) {
#pragma unroll
    for (int e = 0; e < kPer; ++e) put_shared(part + c0 + e, o[e]);
    if (c0 == 0) {
      put_shared(st, top);
      put_shared(st + 1, l);
    }
  }
  // The last workgroup of the sequence's items joins them, a row or two for each wavefront (tickets are given where a
  // sequence has no more rows, which are one piece, and where there are no shared fronts).  Each one's
  // partial results are visible on every die before its ticket is counted; the ticket is a zero again afterwards.
  __shared__ int last_one;
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
  if (threadIdx.x == 0) {
    int* ticket = a.tickets + (static_cast<int64_t>(run.slot) * a.H + h) * kApart;
    last_one = __hip_atomic_fetch_add(ticket, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == run.items - 1;
    if (last_one) __hip_atomic_store(ticket, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
  __syncthreads();
  if (!last_one || wave >= rows) return;
  if (D > 64 || rows <= kWaves) {
    join_rows<D, BF16, 1>(a, run, wave, rows, h);
  } else if constexpr (D == 64) {
    join_rows<D, BF16, 2>(a, run, wave, rows, h);
  }
}

// WAVES wavefronts per (packed row, query head): the items of its sequence's shared front, then its own.  4-5 us: a launch
// and two round trips.
template <int D, bool BF16, int WAVES>
__global__ __launch_bounds__(kThreads) void paged_merge_kernel(DecodeArgs a, int64_t total) {
  const int wave = threadIdx.x >> 6, part = wave % WAVES, lane = threadIdx.x & 63;
  const int64_t at = static_cast<int64_t>(blockIdx.x) * (kWaves / WAVES) + wave / WAVES;
  if (at >= total) return;
  const int Hq = a.H * a.rep;
  const int n = static_cast<int>(at / Hq), head = static_cast<int>(at % Hq), h = head / a.rep;
  // as many sequences as rows, none with two: one of each; without fronts a sequence is the run of its number
  const int longest = a.step[5], count = a.step[8];
  const int i = a.n == 1 ? 0 : longest == 1 && total == static_cast<int64_t>(a.n) * Hq ? n : step_find(a.step, a.n, 3, n);
  const int* runs = step_runs(a.step, a.n);
  const StepRun own = step_run(runs, count == a.n ? i : step_seq(a.step, i).run);
  if (n >= own.row0 + own.tokens) return;
  if (own.items < 2 && !own.front) return;    // its workgroup has written the result
  Join<D, false, 1, (WAVES > 1)> j;
  if (own.front) {
    const StepRun front = step_run(runs, own.front - 1);
    const int R[1] = {(n - front.row0) * a.rep + head % a.rep};
    j.add(a, front, R, h, front.items * part / WAVES, front.items * (part + 1) / WAVES);
  }
  const int R[1] = {(n - own.row0) * a.rep + head % a.rep};
  j.add(a, own, R, h, own.items * part / WAVES, own.items * (part + 1) / WAVES);
  if constexpr (WAVES > 1) {
    __shared__ float sums[kWaves][D], stats[kWaves][2];
#pragma unroll
    for (int e = 0; e < D / 64; ++e) sums[wave][lane * (D / 64) + e] = j.o[0][e];
    if (lane == 0) {
      stats[wave][0] = j.top[0];
      stats[wave][1] = j.l[0];
    }
    __syncthreads();                          // a workgroup is one row: all or none get here
    if (part) return;
    float top = stats[0][0];
#pragma unroll
    for (int i = 1; i < WAVES; ++i) top = fmaxf(top, stats[i][0]);
    const float safe = top == -INFINITY ? 0.0f : top;
    j = Join<D, false, 1, (WAVES > 1)>();
#pragma unroll
    for (int i = 0; i < WAVES; ++i) {
      const float f = __builtin_amdgcn_exp2f(stats[i][0] - safe);
      j.l[0] += f * stats[i][1];
#pragma unroll
      for (int e = 0; e < D / 64; ++e) j.o[0][e] += weigh(f, sums[i][lane * (D / 64) + e]);
    }
  }
  j.template put<BF16>(0, a.out + at * D);
}

int64_t pieces_of(int64_t rep, int64_t tokens) { return (rep * tokens + kRows - 1) / kRows; }

}  // namespace
}  // namespace kvq

using namespace kvq;

extern "C" int64_t kvq_paged_decode_workspace(int64_t split_tokens, int64_t H, int64_t rep, int64_t D) {
  if (split_tokens < 0 || split_tokens >= INT64_C(1) << 31 || H < 1 || rep < 1 || (D != 64 && D != 128)) return -1;
  return split_tokens * rep * H * (D + 2);
}

static int paged_decode(const void* q, int64_t q_st, int64_t q_sh, int dtype, int64_t rows, int64_t Hq, int64_t H, int64_t D,
                                float scaling, const int32_t* step, int64_t sequences, int64_t split_items, int64_t run_tokens,
                                int64_t split_tokens, int joins, const int32_t* table, int64_t max_blocks, int64_t P, int code, const uint8_t* kc, const uint8_t* vc, const float* sc,
                                const void* ko, const void* vo, void* out, float* workspace, int64_t workspace_floats, int32_t* tickets,
                                bool all, void* stream) {
  KVQ_REQUIRE(D == 64 || D == 128, "kvq_paged_decode: head_dim must be 64 or 128 (got %lld)", static_cast<long long>(D));
  KVQ_REQUIRE(P == 32 || P == 64 || P == 128, "kvq_paged_decode: pages hold 32, 64 or 128 tokens");
  KVQ_REQUIRE(dtype == KVQ_F16 || dtype == KVQ_BF16, "kvq_paged_decode: queries must be fp16 or bf16");
  KVQ_REQUIRE(code == kCodeInt8 || code == kCodeE4M3, "kvq_paged_decode: unknown code %d", code);
  KVQ_REQUIRE(H > 0 && Hq > 0 && Hq % H == 0 && rows > 0 && run_tokens > 0 && split_items > 0 && sequences > 0, "kvq_paged_decode: bad sizes");
  KVQ_REQUIRE(q && step && table && kc && vc && sc && ko && vo && out && (workspace || !joins), "kvq_paged_decode: null pointer");
  KVQ_REQUIRE(reinterpret_cast<uintptr_t>(q) % 16 == 0 && (q_st | q_sh) % 8 == 0 && reinterpret_cast<uintptr_t>(out) % 16 == 0 &&
                  reinterpret_cast<uintptr_t>(workspace) % 16 == 0,
              "kvq_paged_decode: rows and strides must be multiples of 16 bytes");
  const int64_t rep = Hq / H, need = joins ? kvq_paged_decode_workspace(split_tokens, H, rep, D) : 0, pieces = pieces_of(rep, run_tokens);
  KVQ_REQUIRE(need >= 0, "kvq_paged_decode: too many split tokens (%lld)", static_cast<long long>(split_tokens));
  KVQ_REQUIRE(workspace_floats >= need, "kvq_paged_decode: workspace of %lld floats, %lld needed", static_cast<long long>(workspace_floats),
              static_cast<long long>(need));
  DecodeArgs a{static_cast<const uint16_t*>(q), q_st, q_sh, step, static_cast<int>(sequences), table, max_blocks,
               static_cast<int>(H), static_cast<int>(rep), static_cast<int>(pieces), scaling * 1.44269504088896341f, kc, vc, sc,
               static_cast<const uint16_t*>(ko), static_cast<const uint16_t*>(vo), static_cast<uint16_t*>(out), workspace,
               split_tokens * rep, all, rep * run_tokens * D <= kWaves * 128 && split_items * H <= 256 && split_items <= 64 * sequences ? tickets : nullptr};
  // Joining in the launch, against a launch for it, in us.  One sequence, 8 KV heads: of 128 and 4096 tokens, 136 workgroups,
  // with one row 9.5 / 11.1, four 10.4 / 11.2, eight 12.6 / 11.2 (a wavefront's rows share its loads past the caches); of 64, four
  // rows 8.0 / 10.2, eight 8.7 / 10.2.  768 workgroups 26.1 / 23.9 (their stores and the wait for the last one); 2 KV heads, 30000
  // tokens, 118 items of one sequence 17.1 / 12.5.
  // The launch takes a workgroup for each row, a quarter of the items to a wavefront, where sequences have many items and
  // the rows are few: those 118 items 22.5 -> 12.5; otherwise a wavefront for each row: 16 sequences of 5 items, 896 rows,
  // 13.9 against 15.0.
  const int64_t blocks = (split_items * H + 7) / 8 * 8 * a.pieces,
                waves = rows * Hq <= 1024 && split_items >= 16 * sequences ? kWaves : 1,
                merges = (rows * Hq * waves + kWaves - 1) / kWaves;
  KVQ_REQUIRE(blocks <= kMaxGrid && merges <= kMaxGrid, "kvq_paged_decode: too many rows");
  auto run = [&](auto d, auto p, auto c, auto t) {
    constexpr int D_ = decltype(d)::value, P_ = decltype(p)::value, C_ = decltype(c)::value;
    constexpr bool T_ = decltype(t)::value != 0;
    hipLaunchKernelGGL((paged_split_kernel<D_, P_, C_, T_>), dim3(static_cast<uint32_t>(blocks)), dim3(kThreads), 0,
                       static_cast<hipStream_t>(stream), a);
    if (a.tickets || !joins) return;
    auto join = [&](auto w) {
      hipLaunchKernelGGL((paged_merge_kernel<D_, T_, decltype(w)::value>), dim3(static_cast<uint32_t>(merges)), dim3(kThreads), 0,
                         static_cast<hipStream_t>(stream), a, rows * Hq);
    };
    if (waves == kWaves) join(std::integral_constant<int, kWaves>{});
    else join(std::integral_constant<int, 1>{});
  };
  using Zero = std::integral_constant<int, 0>;
  using One = std::integral_constant<int, 1>;
  auto by_type = [&](auto d, auto p, auto c) {
    if (dtype == KVQ_BF16) run(d, p, c, One{});
    else run(d, p, c, Zero{});
  };
  auto by_code = [&](auto d, auto p) {
    if (code == kCodeInt8) by_type(d, p, Zero{});
    else by_type(d, p, One{});
  };
  auto by_page = [&](auto d) {
    if (P == 32) by_code(d, std::integral_constant<int, 32>{});
    else if (P == 64) by_code(d, std::integral_constant<int, 64>{});
    else by_code(d, std::integral_constant<int, 128>{});
  };
  if (D == 64) by_page(std::integral_constant<int, 64>{});
  else by_page(std::integral_constant<int, 128>{});
  KVQ_LAUNCH_CHECK("kvq_paged_decode");
  return KVQ_OK;
}

extern "C" int kvq_paged_decode(const void* q, int64_t q_st, int64_t q_sh, int dtype, int64_t rows, int64_t Hq, int64_t H, int64_t D,
                                float scaling, const int32_t* step, int64_t sequences, int64_t split_items, int64_t run_tokens,
                                int64_t split_tokens, int joins, const int32_t* table, int64_t max_blocks, int64_t P, int code, const uint8_t* kc, const uint8_t* vc, const float* sc,
                                const void* ko, const void* vo, void* out, float* workspace, int64_t workspace_floats, int32_t* tickets,
                                void* stream) {
  return paged_decode(q, q_st, q_sh, dtype, rows, Hq, H, D, scaling, step, sequences, split_items, run_tokens, split_tokens, joins, table, max_blocks, P, code, kc, vc, sc, ko, vo, out, workspace, workspace_floats, tickets, false, stream);
}

extern "C" int kvq_paged_decode_held(const void* q, int64_t q_st, int64_t q_sh, int dtype, int64_t rows, int64_t Hq, int64_t H, int64_t D,
                                float scaling, const int32_t* step, int64_t sequences, int64_t split_items, int64_t run_tokens,
                                int64_t split_tokens, int joins, const int32_t* table, int64_t max_blocks, int64_t P, int code, const uint8_t* kc, const uint8_t* vc, const float* sc,
                                const void* ko, const void* vo, void* out, float* workspace, int64_t workspace_floats, int32_t* tickets,
                                int all, void* stream) {
  return paged_decode(q, q_st, q_sh, dtype, rows, Hq, H, D, scaling, step, sequences, split_items, run_tokens, split_tokens, joins, table, max_blocks, P, code, kc, vc, sc, ko, vo, out, workspace, workspace_floats, tickets, all != 0, stream);
}
