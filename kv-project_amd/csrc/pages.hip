// The paged 8-bit cache: its page accounts (host), filling it, reading it back and moving its pages.
//
// A block is coded once, when its last token comes: a = max(|x|, 2^-100) over the P x D values of one KV
// head, scale = a * (1 / top), code = rne(x * ((1 / a) * top)), top = 127 (int8) or 448 (e4m3), each
// operation rounded to float32 (as torch divides by a number, and a number by a tensor, on this device;
// bf16 values meet exact ties often enough for the last bit to count).  The codes of a block therefore do not depend
// on how its tokens arrived.  A block that holds an infinity or a NaN gets the scale NaN: its tokens read as NaN.
//
// All of these kernels move bytes: filling reads 4 D and writes 2 D bytes per token and KV head, reading back the
// reverse.  16 prompts of 6001 to 8200 tokens, 8 KV heads of 128: filling 129-144 us for 694 MB (4.8-5.4 TB/s), reading
// back 116-123 (5.6-6.0); a large copy reaches 4.9.  A few tokens: 2-5 us each, a launch and its round trips.
#include <algorithm>
#include <cmath>
#include <cstring>

#include "mfma_common.hpp"
#include "pages.hpp"

namespace kvq {
namespace {

constexpr int kThreads = 256;
constexpr int kWords = 960;                   // words that go with a launch by value

struct WordBlock {
  int w[kWords];
};

__global__ __launch_bounds__(kThreads) void write_words_kernel(WordBlock b, int* dst, int n) {
  for (int i = threadIdx.x; i < n; i += kThreads) dst[i] = b.w[i];
}

int write_words(const int32_t* src, int64_t n, int32_t* dst, hipStream_t stream) {
  for (int64_t at = 0; at < n; at += kWords) {
    WordBlock b;
    const int m = static_cast<int>(n - at < kWords ? n - at : kWords);
    memcpy(b.w, src + at, sizeof(int) * m);
    hipLaunchKernelGGL(write_words_kernel, dim3(1), dim3(kThreads), 0, stream, b, dst + at, m);
  }
  KVQ_LAUNCH_CHECK("kvq_pages: step description");
  return KVQ_OK;
}

// The heads of one block on one of the 8 dies: their rows lie next to each other in memory.
struct BlockHead {
  int item, h;
};
__device__ __forceinline__ BlockHead block_head(int H) {
  const int i = blockIdx.x / 8;
  return {i / H * 8 + static_cast<int>(blockIdx.x % 8), i % H};
}
int64_t block_grid(int64_t items, int64_t H) { return (items + 7) / 8 * 8 * H; }

// ---- filling ----------------------------------------------------------------------------------

struct Rows16 {                               // packed rows (n, H, D) of 16-bit elements
  const uint16_t* p;
  int64_t st, sh;
};

template <bool BF16>
__device__ __forceinline__ float to_f32(uint32_t h) {
  if constexpr (BF16) return __uint_as_float(h << 16);
  else return f16_to_f32(static_cast<uint16_t>(h));
}

// |x| of both halves as bit patterns: ordered as unsigned numbers, infinities and NaN on top
__device__ __forceinline__ uint32_t abs_max2(uint32_t m, uint32_t w) {
  const uint32_t a = w & 0x7fffu, b = (w >> 16) & 0x7fffu;
  m = m > a ? m : a;
  return m > b ? m : b;
}

// Four values of at most the type's top as codes, rounded to nearest even.  int8: 1.5 2^23 + x is a float32 whose
// low byte is the rounded x.
template <int CODE>
__device__ __forceinline__ uint32_t encode4(float a, float b, float c, float d) {
#pragma clang fp contract(off)
  if constexpr (CODE == kCodeInt8) {
    const uint32_t x = __float_as_uint(a + 12582912.0f), y = __float_as_uint(b + 12582912.0f);
    const uint32_t z = __float_as_uint(c + 12582912.0f), w = __float_as_uint(d + 12582912.0f);
    return __builtin_amdgcn_perm(__builtin_amdgcn_perm(w, z, 0x0c0c0400u), __builtin_amdgcn_perm(y, x, 0x0c0c0400u), 0x05040100u);
  } else {
    int r = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
    return static_cast<uint32_t>(__builtin_amdgcn_cvt_pk_fp8_f32(c, d, r, true));
  }
}

struct Scale {
  float scale, inv;
};

// scale and its inverse from the largest |bits| of a block; a block with an infinity or a NaN is marked
// by the scale NaN, its codes are zeros
template <int CODE, bool BF16>
__device__ __forceinline__ Scale block_scale(uint32_t bits) {
  constexpr float top = CODE == kCodeInt8 ? 127.0f : 448.0f;
  const float a = fmaxf(to_f32<BF16>(bits), 0x1p-100f);
  if (bits >= (BF16 ? 0x7f80u : 0x7c00u)) return {__uint_as_float(0x7fc00000u), 0.0f};
  return {a * (1.0f / top), __fdiv_rn(1.0f, a) * top};
}

// One workgroup per (item, KV head).  Keys and values of the block are held in registers (16 bytes a
// load), the largest magnitudes reduced over the workgroup, and the codes written; values turn to
// channel-major order through LDS.  A block that stays open is copied to the open buffer instead.
template <int D, int P, int CODE, bool BF16>
__global__ __launch_bounds__(kThreads) void append_kernel(Rows16 k, Rows16 v, const int* __restrict__ step, int* __restrict__ table,
                                                          int64_t max_blocks, int H, uint8_t* __restrict__ kc,
                                                          uint8_t* __restrict__ vc, float* __restrict__ sc,
                                                          uint16_t* __restrict__ ko, uint16_t* __restrict__ vo) {
  constexpr int kChunks = P * D / 8, kPer = kChunks / kThreads;      // pieces of 8 elements, per thread
  constexpr int kRow = D / 8;                                       // pieces of a token
  // values turn to channel-major order in LDS: channel c's tokens 8 u .. at piece u ^ (c / 8) of its row, which spreads the
  // channels of a wavefront's writes (8 apart) over P / 8 places; with 128 channels two of them still share the banks
  // at 64 tokens, four at 32 (31 conflict cycles a wavefront, 1.8 million of a large fill of 144 us)
  __shared__ __align__(16) uint16_t turn[D * P];
  auto place = [](int c, int t) { return c * P + (((t >> 3) ^ (c >> 3)) & (P / 8 - 1)) * 8 + (t & 7); };
  __shared__ uint32_t top[8];
  const BlockHead bh = block_head(H);
  const int item = bh.item, h = bh.h, tid = threadIdx.x;
  const int n = step[0];
  if (item >= step[1]) return;
  const StepSeq s = step_seq(step, step[4] ? item : step_find(step, n, 4, item));
  const int j = s.pos0 / P + item - s.item0;                        // block of the sequence
  const int first = j * P, end = s.pos0 + s.count;
  const int from = first > s.pos0 ? first : s.pos0;                 // tokens [from, to) of the block are new
  const int to = first + P < end ? first + P : end;
  const int64_t open_before = (static_cast<int64_t>(s.slot) * 2 + (s.bufs & 1)) * H + h;
  const int64_t open_after = (static_cast<int64_t>(s.slot) * 2 + (s.bufs >> 1 & 1)) * H + h;
  const int64_t row0 = s.row0 - s.pos0;                             // packed row of a token: row0 + position
  const uint16_t* kn = k.p + h * k.sh;
  const uint16_t* vn = v.p + h * v.sh;

  if (to < first + P) {                                             // stays open: new rows into the open buffer
    uint16_t* kd = ko + open_after * P * D;
    uint16_t* vd = vo + open_after * P * D;
    const int rows = to - from;
    for (int i = tid; i < rows * kRow; i += kThreads) {
      const int t = i / kRow, c = i % kRow * 8;
      const int64_t at = row0 + from + t;
      *reinterpret_cast<uint4*>(kd + (from - first + t) * D + c) = *reinterpret_cast<const uint4*>(kn + at * k.st + c);
      const uint4 w = *reinterpret_cast<const uint4*>(vn + at * v.st + c);
      const uint32_t ws[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
      for (int e = 0; e < 8; ++e)
        vd[(c + e) * P + from - first + t] = static_cast<uint16_t>(ws[e >> 1] >> (16 * (e & 1)));
    }
    return;
  }

  // the whole block: rows before `from` out of the open buffer
  const uint16_t* kb = ko + open_before * P * D;
  const uint16_t* vb = vo + open_before * P * D;
  uint4 kw[kPer];
  uint32_t kmax = 0, vmax = 0;
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const int q = tid + i * kThreads, t = q / kRow, c = q % kRow * 8;
    const bool fresh = first + t >= from;
    kw[i] = *reinterpret_cast<const uint4*>(fresh ? kn + (row0 + first + t) * k.st + c : kb + t * D + c);
  }
  const int old = from - first;                                     // tokens that lie in the open buffer
  if (old == 0) {
    constexpr int kPairs = (kPer + 1) / 2;                          // two tokens at a time: words of a channel's pair
    uint4 vx[kPairs], vy[kPairs];
#pragma unroll
    for (int i = 0; i < kPairs; ++i) {                              // all on their way before the first is used, the keys too
      const int q = tid + i * kThreads, t = q / kRow * 2, c = q % kRow * 8;
      const uint16_t* at = vn + (row0 + first + t) * v.st + c;
      if (kPer % 2 == 0 || q < kChunks / 2) {
        vx[i] = *reinterpret_cast<const uint4*>(at);
        vy[i] = *reinterpret_cast<const uint4*>(at + v.st);
      }
    }
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int i = 0; i < kPairs; ++i) {
      const int q = tid + i * kThreads, t = q / kRow * 2, c = q % kRow * 8;
      if (kPer % 2 && q >= kChunks / 2) break;
      const uint4 x = vx[i], y = vy[i];
      const uint32_t xs[4] = {x.x, x.y, x.z, x.w}, ys[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
      for (int e = 0; e < 8; ++e)
        *reinterpret_cast<uint32_t*>(turn + place(c + e, t)) = __builtin_amdgcn_perm(ys[e >> 1], xs[e >> 1], e & 1 ? 0x07060302u : 0x05040100u);
    }
  } else {
    for (int i = tid; i < (P - old) * kRow; i += kThreads) {
      const int t = old + i / kRow, c = i % kRow * 8;
      const uint4 w = *reinterpret_cast<const uint4*>(vn + (row0 + first + t) * v.st + c);
      const uint32_t ws[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
      for (int e = 0; e < 8; ++e) turn[place(c + e, t)] = static_cast<uint16_t>(ws[e >> 1] >> (16 * (e & 1)));
    }
    for (int i = tid; i < D * (P / 8); i += kThreads) {             // pieces of 8 tokens, the last one in part
      const int c = i / (P / 8), t = i % (P / 8) * 8;
      if (t + 8 <= old) {
        *reinterpret_cast<uint4*>(turn + place(c, t)) = *reinterpret_cast<const uint4*>(vb + c * P + t);
      } else {
        for (int e = 0; e < 8 && t + e < old; ++e) turn[place(c, t + e)] = vb[c * P + t + e];
      }
    }
  }
#pragma unroll
  for (int i = 0; i < kPer; ++i) kmax = abs_max2(abs_max2(abs_max2(abs_max2(kmax, kw[i].x), kw[i].y), kw[i].z), kw[i].w);
  __syncthreads();
  uint4 vw[kPer];                                                   // pieces of 8 tokens of a channel
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const int q = tid + i * kThreads, c = q / (P / 8), t = q % (P / 8) * 8;
    vw[i] = *reinterpret_cast<const uint4*>(turn + place(c, t));
    vmax = abs_max2(abs_max2(abs_max2(abs_max2(vmax, vw[i].x), vw[i].y), vw[i].z), vw[i].w);
  }
  for (int o = 32; o; o >>= 1) {
    const uint32_t a = __shfl_xor(kmax, o), e = __shfl_xor(vmax, o);
    kmax = kmax > a ? kmax : a;
    vmax = vmax > e ? vmax : e;
  }
  if ((tid & 63) == 0) {
    top[tid >> 6] = kmax;
    top[4 + (tid >> 6)] = vmax;
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    kmax = kmax > top[i] ? kmax : top[i];
    vmax = vmax > top[4 + i] ? vmax : top[4 + i];
  }
  const Scale ks = block_scale<CODE, BF16>(kmax), vs = block_scale<CODE, BF16>(vmax);
  const int page = step[step[9] + item];
  const int64_t at = (static_cast<int64_t>(page) * H + h) * P * D;
  if (tid == 0) {
    float2* p = reinterpret_cast<float2*>(sc) + static_cast<int64_t>(page) * H + h;
    *p = make_float2(ks.scale, vs.scale);
    if (h == 0) table[s.slot * max_blocks + j] = page;
  }
  auto put = [&](uint8_t* dst, const uint4& w, const Scale& z) {
#pragma clang fp contract(off)                                      // the product is rounded before it is rounded to a code
    const bool bad = z.inv == 0.0f;                                 // 0 * inf would be a NaN code
    const uint32_t ws[4] = {bad ? 0 : w.x, bad ? 0 : w.y, bad ? 0 : w.z, bad ? 0 : w.w};
    float x[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = to_f32<BF16>(ws[e >> 1] >> (16 * (e & 1)) & 0xffffu) * z.inv;
    *reinterpret_cast<uint2*>(dst) = make_uint2(encode4<CODE>(x[0], x[1], x[2], x[3]), encode4<CODE>(x[4], x[5], x[6], x[7]));
  };
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const int q = tid + i * kThreads;
    put(kc + at + q * 8, kw[i], ks);
    put(vc + at + q * 8, vw[i], vs);
  }
}

// ---- reading back -----------------------------------------------------------------------------

template <int CODE>
__device__ __forceinline__ float decode1(uint32_t w, int e) {
  if constexpr (CODE == kCodeInt8) return static_cast<float>(static_cast<int8_t>(w >> (8 * e)));
  else
    return e == 0   ? __builtin_amdgcn_cvt_f32_fp8(static_cast<int>(w), 0)
           : e == 1 ? __builtin_amdgcn_cvt_f32_fp8(static_cast<int>(w), 1)
           : e == 2 ? __builtin_amdgcn_cvt_f32_fp8(static_cast<int>(w), 2)
                    : __builtin_amdgcn_cvt_f32_fp8(static_cast<int>(w), 3);
}

template <bool BF16>
__device__ __forceinline__ uint16_t from_f32(float x) {
  if constexpr (BF16) return f32_to_bf16(x);
  else return f32_to_f16(x);
}

// Whole sequences by value with the launch: {slot, tokens, first row, first block, open buffer} of each
constexpr int kWhole = 5, kMostWhole = kWords / kWhole;

// One workgroup per (block, KV head): dense rows (rows, H, D) of keys and values.
template <int D, int P, int CODE, bool BF16>
__global__ __launch_bounds__(kThreads) void rows_kernel(WordBlock whole, int n, int blocks, const int* __restrict__ table, int64_t max_blocks,
                                                        int H, const uint8_t* __restrict__ kc, const uint8_t* __restrict__ vc,
                                                        const float* __restrict__ sc, const uint16_t* __restrict__ ko,
                                                        const uint16_t* __restrict__ vo, uint16_t* __restrict__ k_out,
                                                        uint16_t* __restrict__ v_out) {
  constexpr int kChunks = P * D / 8, kPer = kChunks / kThreads, kRow = D / 8;
  constexpr int kPitch = D + 8;
  __shared__ __align__(16) uint16_t turn[P * kPitch];
  const BlockHead bh = block_head(H);
  const int item = bh.item, h = bh.h, tid = threadIdx.x;
  if (item >= blocks) return;
  const int lo = __builtin_amdgcn_readfirstlane(last_not_above(whole.w + 3, kWhole, n, item));
  const int* s = whole.w + kWhole * lo;
  const int64_t slot = s[0];
  const int j = item - s[3], first = j * P;
  const int rows = s[1] - first < P ? s[1] - first : P;
  const bool open = rows < P;
  const int64_t out = (static_cast<int64_t>(s[2] + first) * H + h) * D;
  int64_t at;
  float2 z = make_float2(1.0f, 1.0f);
  if (open) {
    at = ((slot * 2 + s[4]) * H + h) * P * D;
  } else {
    const int64_t page = table[slot * max_blocks + j];
    at = (page * H + h) * P * D;
    z = reinterpret_cast<const float2*>(sc)[page * H + h];
  }
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const int q = tid + i * kThreads, c = q / (P / 8), t = q % (P / 8) * 8;
    if (open) {
      const uint4 w = *reinterpret_cast<const uint4*>(vo + at + q * 8);
      const uint32_t ws[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
      for (int e = 0; e < 8; ++e) turn[(t + e) * kPitch + c] = static_cast<uint16_t>(ws[e >> 1] >> (16 * (e & 1)));
    } else {
      const uint2 w = *reinterpret_cast<const uint2*>(vc + at + q * 8);
#pragma unroll
      for (int e = 0; e < 8; ++e) turn[(t + e) * kPitch + c] = from_f32<BF16>(decode1<CODE>(e < 4 ? w.x : w.y, e & 3) * z.y);
    }
  }
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const int q = tid + i * kThreads, t = q / kRow, c = q % kRow * 8;
    if (t >= rows) continue;
    uint4 o;
    if (open) {
      o = *reinterpret_cast<const uint4*>(ko + at + q * 8);
    } else {
      const uint2 w = *reinterpret_cast<const uint2*>(kc + at + q * 8);
      uint32_t r[4];
#pragma unroll
      for (int e = 0; e < 4; ++e)
        r[e] = from_f32<BF16>(decode1<CODE>(e < 2 ? w.x : w.y, 2 * e & 3) * z.x) |
               static_cast<uint32_t>(from_f32<BF16>(decode1<CODE>(e < 2 ? w.x : w.y, (2 * e + 1) & 3) * z.x)) << 16;
      o = make_uint4(r[0], r[1], r[2], r[3]);
    }
    *reinterpret_cast<uint4*>(k_out + out + static_cast<int64_t>(t) * H * D + c) = o;
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const int q = tid + i * kThreads, t = q / kRow, c = q % kRow * 8;
    if (t >= rows) continue;
    *reinterpret_cast<uint4*>(v_out + out + static_cast<int64_t>(t) * H * D + c) = *reinterpret_cast<const uint4*>(turn + t * kPitch + c);
  }
}

// ---- forking and moving -----------------------------------------------------------------------

// {source slot, open buffer, destination slot, tokens} of each pair
struct ForkPairs {
  int w[kWords];
};

// Workgroup (pair, layer * H + h): the open rows of that head; the first of a pair copies the table row.
__global__ __launch_bounds__(kThreads) void fork_kernel(ForkPairs f, int* table, int64_t max_blocks, int64_t slots, int H, int P, int D,
                                                        uint16_t* ko, uint16_t* vo) {
  const int* e = f.w + 4 * blockIdx.x;
  const int64_t src = e[0], dst = e[2];
  const int len = e[3], r = len % P, tid = threadIdx.x;
  if (blockIdx.y == 0)
    for (int i = tid; i < len / P; i += kThreads) table[dst * max_blocks + i] = table[src * max_blocks + i];
  const int64_t layer = blockIdx.y / H, h = blockIdx.y % H;
  const int64_t from = (((layer * slots + src) * 2 + e[1]) * H + h) * P * D, to = ((layer * slots + dst) * 2 * H + h) * P * D;
  for (int i = tid; i < r * D / 8; i += kThreads)
    *reinterpret_cast<uint4*>(ko + to + i * 8) = *reinterpret_cast<const uint4*>(ko + from + i * 8);
  const int pieces = (r + 7) / 8;                                   // of 8 tokens of a channel
  for (int i = tid; i < pieces * D; i += kThreads) {
    const int64_t at = i / pieces * P + i % pieces * 8;
    *reinterpret_cast<uint4*>(vo + to + at) = *reinterpret_cast<const uint4*>(vo + from + at);
  }
}

struct Pool {
  uint8_t *kc, *vc;
  float* sc;
};

// {from, to} of each page
struct Moves {
  int w[kWords];
};

// Workgroup (move, layer): one page with all its heads, which lie behind one another (keys and values 64 KB each at 8
// heads of 128 and 64 tokens).  The pages of 12 sequences in 32 layers, 3.8 GB read and written: 727-740 us, 5.2 TB/s.
__global__ __launch_bounds__(kThreads) void move_kernel(Moves m, Pool s, Pool d, int64_t s_pages, int64_t d_pages, int H, int64_t page_bytes) {
  const int64_t layer = blockIdx.y, from = layer * s_pages + m.w[2 * blockIdx.x], to = layer * d_pages + m.w[2 * blockIdx.x + 1];
  const uint4* a = reinterpret_cast<const uint4*>(s.kc + from * page_bytes);
  const uint4* b = reinterpret_cast<const uint4*>(s.vc + from * page_bytes);
  uint4* x = reinterpret_cast<uint4*>(d.kc + to * page_bytes);
  uint4* y = reinterpret_cast<uint4*>(d.vc + to * page_bytes);
  for (int64_t i = threadIdx.x; i < page_bytes / 16; i += kThreads) {
    x[i] = a[i];
    y[i] = b[i];
  }
  for (int i = threadIdx.x; i < 2 * H; i += kThreads) d.sc[to * 2 * H + i] = s.sc[from * 2 * H + i];
}

// entries of the table that name a page behind the new end: those in use are written again by patch_kernel
__global__ __launch_bounds__(kThreads) void clip_kernel(int* __restrict__ table, int64_t n, int pages) {
  const int64_t i = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x;
  if (i < n && table[i] >= pages) table[i] = 0;
}

// {slot, block, page}
struct Patches {
  int w[kWords];
};
__global__ __launch_bounds__(kThreads) void patch_kernel(Patches p, int n, int* __restrict__ table, int64_t max_blocks) {
  for (int i = threadIdx.x; i < n; i += kThreads) table[p.w[3 * i] * max_blocks + p.w[3 * i + 1]] = p.w[3 * i + 2];
}

// ---- the accounts (host) ----------------------------------------------------------------------

// Units of a sequence: those of its full blocks, and those of its open one
int64_t units_of(int64_t len, int64_t page) {
  const int64_t full = len / page * page;
  return (full + kUnit - 1) / kUnit + (len - full + kUnit - 1) / kUnit;
}

// Pages in front that slots a and b share, of the first `most`
int64_t shared(const int32_t* table, int64_t max_blocks, int64_t a, int64_t b, int64_t most) {
  int64_t i = 0;
  while (i < most && table[a * max_blocks + i] == table[b * max_blocks + i]) ++i;
  return i;
}

// A front is worth a run of its own from this many units on: one for each wavefront of a workgroup.
constexpr int64_t kFront = 4;
constexpr int64_t kUneven = 16;

// Fills the description from lens (before), counts and open buffers; pages are written by the caller.  split_cap bounds
// the split items (those of a front weighted by the workgroups that its rows take at four query heads per KV head: the real
// number is not known here, with one or eight of them the weight is four times too large or half).
// With few_cap, the workgroups that have a CU each: of no more than few_units units there are few_cap items, unless that
// makes the longest one more than twice an even share, or there are more sequences and long ones among them; and up to twice split_cap where the longest item is kUneven units
// and 1.5 times an even share at least, and all sequences start at once (8 KV heads of 128: 64 sequences of 100 to 4000
// tokens 61 -> 54 us, but 64 of 3000 to 4000 94 -> 98, and 256 of 16 to 3000 with 16 rows each 187 -> 209).  More sequences
// than places are one item each, however long: 64 of 1000 tokens beside one of 32768 wait for its 513 units, 16 with 63.
// most_run, most_tokens: where the step has to fit a launch that was captured; fronts that do not are left out.
void describe(const int64_t* lens, const uint8_t* open, const int32_t* table, int64_t max_blocks, int64_t page, const int64_t* seq,
              const int64_t* counts, int64_t n, int64_t split_cap, int64_t few_cap, int64_t few_units, int64_t most_run, int64_t most_tokens,
              int32_t* desc) {
  int64_t row = 0, item = 0, longest = 0;
  bool even = true;
  for (int64_t i = 0; i < n; ++i) {
    int32_t* e = desc + kStepHead + kStepSeq * i;
    const int64_t s = seq[i], pos0 = lens[s], count = counts[i], end = pos0 + count;
    const int src = open[s] & 1, dst = pos0 % page && end / page > pos0 / page && end % page ? src ^ 1 : src;
    e[0] = static_cast<int32_t>(s);
    e[1] = static_cast<int32_t>(pos0);
    e[2] = static_cast<int32_t>(count);
    e[3] = static_cast<int32_t>(row);
    e[4] = static_cast<int32_t>(item);
    e[6] = src | dst << 1;
    row += count;
    longest = count > longest ? count : longest;
    item += count ? (end - 1) / page - pos0 / page + 1 : 0;
    even = even && item == i + 1;
  }
  int32_t* last = desc + kStepHead + kStepSeq * n;
  memset(last, 0, sizeof(int32_t) * kStepSeq);
  last[3] = static_cast<int32_t>(row);
  last[4] = static_cast<int32_t>(item);
  int32_t* runs = desc + kStepHead + kStepSeq * (n + 1);
  for (int fronts = 1; fronts >= 0; --fronts) {
    int64_t nr = 0, widest = longest;
    auto add = [&](int64_t slot, int64_t row0, int64_t tokens, int64_t u0, int64_t u1, int64_t b) {
      int32_t* r = runs + kStepRun * nr++;
      r[0] = static_cast<int32_t>(slot);
      r[1] = static_cast<int32_t>(row0);
      r[2] = static_cast<int32_t>(tokens);
      r[3] = static_cast<int32_t>(u0);
      r[4] = static_cast<int32_t>(tokens ? u1 : u0);
      r[7] = static_cast<int32_t>(b);
      const int32_t* e = desc + kStepHead + kStepSeq * (b < 0 ? 0 : b);
      r[8] = b < 0 ? 0 : e[1];
      r[9] = b < 0 ? 0 : e[6] >> 1;
      r[10] = b < 0 ? 0 : e[7];
    };
    for (int64_t i = 0; i < n;) {
      int64_t j = i + 1, common = 0, tokens = counts[i];
      for (; fronts && counts[i] && j < n && counts[j]; ++j) {
        const int64_t a = lens[seq[i]] / page, b = lens[seq[j]] / page, most = a < b ? a : b;
        const int64_t c = shared(table, max_blocks, seq[i], seq[j], j > i + 1 && common < most ? common : most);
        if (c * page < kFront * kUnit || 2 * c < common) break;
        common = c;
        tokens += counts[j];
      }
      const int64_t front = j > i + 1 ? common * page / kUnit : 0;
      if (front) add(seq[i], desc[kStepHead + kStepSeq * i + 3], tokens, 0, front, -1);
      widest = front && tokens > widest ? tokens : widest;
      const int64_t of = front ? nr : 0;      // 1 + its index
      for (int64_t b = i; b < j; ++b) {
        int32_t* e = desc + kStepHead + kStepSeq * b;
        e[5] = static_cast<int32_t>(nr);
        e[7] = static_cast<int32_t>(of);
        add(seq[b], e[3], counts[b], front, units_of(lens[seq[b]] + counts[b], page), b);
      }
      i = j;
    }
    int64_t most = 4;                         // a wavefront takes a unit at least
    for (int64_t i = 0; i < nr; ++i) most = runs[kStepRun * i + 4] - runs[kStepRun * i + 3] > most ? runs[kStepRun * i + 4] - runs[kStepRun * i + 3] : most;
    auto splits = [&](int64_t i, int64_t per) { return (runs[kStepRun * i + 4] - runs[kStepRun * i + 3] + per - 1) / per; };
    auto weighted = [&](int64_t per) {
      int64_t w = 0;
      for (int64_t i = 0; i < nr; ++i) w += splits(i, per) * (runs[kStepRun * i + 7] < 0 ? (runs[kStepRun * i + 2] + 3) / 4 : 1);
      return w;
    };
    auto units = [&](int64_t cap) {           // of an item, so that there are at most `cap` items
      int64_t lo = 4, hi = most;
      while (lo < hi) {
        const int64_t mid = (lo + hi) / 2;
        if (weighted(mid) <= cap) hi = mid;
        else lo = mid + 1;
      }
      return lo;
    };
    int64_t lo = units(split_cap), cap = split_cap;
    const int64_t all = weighted(1), active = std::count_if(counts, counts + n, [](int64_t c) { return c > 0; });
    auto even_share = [&](int64_t items) { const int64_t x = (all + items - 1) / items; return x > 4 ? x : 4; };
    const int64_t few = few_cap > 0 && few_cap < split_cap && all <= few_units ? units(few_cap) : 0;
    if (few && few <= 2 * even_share(few_cap) && (few < kUneven || weighted(few) <= few_cap)) {
      lo = few;
    } else if (lo >= kUneven && active <= 2 * few_cap && 2 * lo > 3 * even_share(split_cap)) {
      cap = 2 * split_cap;
      lo = units(cap);
    }
    int64_t split = 0, base = 0;
    bool ones = true, joins = nr > n;
    for (int64_t i = 0; i < nr; ++i) {
      int32_t* r = runs + kStepRun * i;
      r[5] = static_cast<int32_t>(split);
      r[6] = static_cast<int32_t>(base);
      r[11] = static_cast<int32_t>(splits(i, lo));
      split += splits(i, lo);
      base += splits(i, lo) * r[2];
      ones = ones && splits(i, lo) == 1;
      joins = joins || splits(i, lo) > 1;
    }
    if (fronts && nr > n && (weighted(lo) > cap || widest > most_run || base > most_tokens)) continue;
    int32_t* r = runs + kStepRun * nr;
    memset(r, 0, sizeof(int32_t) * kStepRun);
    r[5] = static_cast<int32_t>(split);
    r[6] = static_cast<int32_t>(base);
    desc[0] = static_cast<int32_t>(n);
    desc[1] = static_cast<int32_t>(item);
    desc[2] = static_cast<int32_t>(split);
    desc[3] = static_cast<int32_t>(lo);
    desc[4] = even;
    desc[5] = static_cast<int32_t>(longest);
    desc[6] = static_cast<int32_t>(widest);
    desc[7] = base < INT64_C(1) << 31 ? static_cast<int32_t>(base) : -1;
    desc[8] = static_cast<int32_t>(nr);
    desc[9] = static_cast<int32_t>(kStepHead + kStepSeq * (n + 1) + kStepRun * (nr + 1));
    desc[10] = joins;
    desc[11] = ones;
    last[5] = static_cast<int32_t>(nr);
    return;
  }
}

int64_t item_cap(int64_t page, const int64_t* counts, int64_t n) {
  int64_t cap = 0;                                                  // blocks that counts[i] tokens touch at most
  for (int64_t i = 0; i < n; ++i) cap += counts[i] ? (counts[i] + page - 2) / page + 1 : 0;
  return cap;
}

bool page_ok(int64_t P, int64_t D) { return (P == 32 || P == 64 || P == 128) && (D == 64 || D == 128); }

}  // namespace
}  // namespace kvq

using namespace kvq;

#define KVQ_PAGES_DISPATCH(...)                                                                                  \
  auto run_ = [&](auto d_, auto p_, auto c_, auto t_) {                                                           \
    constexpr int D_ = decltype(d_)::value, P_ = decltype(p_)::value, C_ = decltype(c_)::value;                   \
    constexpr bool T_ = decltype(t_)::value != 0;                                                                 \
    __VA_ARGS__;                                                                                                  \
  };                                                                                                              \
  auto by_t_ = [&](auto d_, auto p_, auto c_) {                                                                   \
    if (dtype == KVQ_BF16) run_(d_, p_, c_, std::integral_constant<int, 1>{});                                    \
    else run_(d_, p_, c_, std::integral_constant<int, 0>{});                                                      \
  };                                                                                                              \
  auto by_c_ = [&](auto d_, auto p_) {                                                                            \
    if (code == kCodeInt8) by_t_(d_, p_, std::integral_constant<int, 0>{});                                       \
    else by_t_(d_, p_, std::integral_constant<int, 1>{});                                                         \
  };                                                                                                              \
  auto by_p_ = [&](auto d_) {                                                                                     \
    if (P == 32) by_c_(d_, std::integral_constant<int, 32>{});                                                    \
    else if (P == 64) by_c_(d_, std::integral_constant<int, 64>{});                                               \
    else by_c_(d_, std::integral_constant<int, 128>{});                                                           \
  };                                                                                                              \
  if (D == 64) by_p_(std::integral_constant<int, 64>{});                                                          \
  else by_p_(std::integral_constant<int, 128>{});

#define KVQ_PAGES_REQUIRE(what)                                                                                     \
  KVQ_REQUIRE(page_ok(P, D), what ": head_dim must be 64 or 128 and the page 32, 64 or 128 tokens (got %lld, %lld)", \
              static_cast<long long>(D), static_cast<long long>(P));                                                \
  KVQ_REQUIRE(code == kCodeInt8 || code == kCodeE4M3, what ": unknown code %d", code);                              \
  KVQ_REQUIRE(dtype == KVQ_F16 || dtype == KVQ_BF16, what ": rows must be fp16 or bf16");                           \
  KVQ_REQUIRE(H > 0 && H < 65536, what ": bad head count");

extern "C" int64_t kvq_pages_step_words(int64_t page, const int64_t* counts, int64_t n) {
  if (n < 0 || (n && !counts) || (page != 32 && page != 64 && page != 128)) return -1;
  for (int64_t i = 0; i < n; ++i)
    if (counts[i] < 0 || counts[i] >= INT64_C(1) << 31) return -1;
  return kStepHead + kStepSeq * (n + 1) + item_cap(page, counts, n) + kStepRun * (2 * n + 1);
}

extern "C" int kvq_pages_extend(int64_t* lens, int32_t* table, int32_t* refs, uint8_t* open, int64_t* account, int64_t slots,
                                int64_t pages, int64_t max_blocks, int64_t page, int64_t max_tokens, const int64_t* seq,
                                const int64_t* counts, int64_t n, int64_t split_cap, int64_t few_cap, int64_t few_units, int64_t most_run,
                                int64_t most_tokens, int32_t* desc, int64_t desc_words, int32_t* desc_device, void* stream) {
  KVQ_REQUIRE(lens && table && refs && open && account && desc && n > 0 && seq && counts,
              "kvq_pages_extend: null pointer or no sequence");
  const int64_t need_words = kvq_pages_step_words(page, counts, n);
  KVQ_REQUIRE(need_words >= 0 && need_words <= desc_words, "kvq_pages_extend: bad counts or a short description");
  int64_t active = 0;
  for (int64_t i = 0; i < n; ++i) active += counts[i] > 0;
  KVQ_REQUIRE(split_cap >= active, "kvq_pages_extend: at least one split item per sequence is needed");
  // every check first: nothing is changed by a call that is refused
  int64_t need = 0, rows = 0, bad = -1, twice = -1;
  int64_t checked = 0;
  for (; checked < n; ++checked) {
    const int64_t s = seq[checked], c = counts[checked];
    if (s < 0 || s >= slots) { bad = checked; break; }
    if (lens[s] < 0) { twice = s; break; }
    if (lens[s] + c > max_tokens) { bad = checked; break; }
    need += (lens[s] + c) / page - lens[s] / page;
    rows += c;
    lens[s] = -lens[s] - 1;                                         // marked as seen
  }
  for (int64_t i = 0; i < checked; ++i) lens[seq[i]] = -lens[seq[i]] - 1;
  KVQ_REQUIRE(twice < 0, "kvq_pages_extend: slot %lld is named twice", static_cast<long long>(twice));
  if (bad >= 0) {
    const int64_t s = seq[bad];
    KVQ_REQUIRE(s >= 0 && s < slots, "kvq_pages_extend: no slot %lld (of %lld)", static_cast<long long>(s), static_cast<long long>(slots));
    KVQ_REQUIRE(false, "decode buffer exhausted: slot %lld holds %lld tokens of %lld, %lld more asked for", static_cast<long long>(s),
                static_cast<long long>(lens[s]), static_cast<long long>(max_tokens), static_cast<long long>(counts[bad]));
  }
  KVQ_REQUIRE(rows < INT64_C(1) << 31, "kvq_pages_extend: too many rows");
  KVQ_REQUIRE(need <= account[0], "decode buffer exhausted: %lld pages needed, %lld free", static_cast<long long>(need),
              static_cast<long long>(account[0]));
  describe(lens, open, table, max_blocks, page, seq, counts, n, split_cap, few_cap, few_units, most_run, most_tokens, desc);
  int32_t* page_of = desc + desc[9];
  int64_t low = account[1];
  for (int64_t i = 0; i < n; ++i) {
    const int32_t* e = desc + kStepHead + kStepSeq * i;
    const int64_t s = seq[i], end = lens[s] + counts[i];
    for (int64_t j = lens[s] / page; counts[i] && j <= (end - 1) / page; ++j) {
      int32_t id = -1;
      if ((j + 1) * page <= end) {
        while (low < pages && refs[low]) ++low;                     // the lowest free page
        KVQ_REQUIRE(low < pages, "kvq_pages_extend: the accounts are broken");
        id = static_cast<int32_t>(low);
        refs[low++] = 1;
        table[s * max_blocks + j] = id;
      }
      page_of[e[4] + j - lens[s] / page] = id;
    }
    open[s] = static_cast<uint8_t>(e[6] >> 1 & 1);
    lens[s] = end;
  }
  account[0] -= need;
  account[1] = low;
  const int64_t words = desc[9] + desc[1];
  return desc_device ? write_words(desc, words, desc_device, static_cast<hipStream_t>(stream)) : KVQ_OK;
}

extern "C" int kvq_pages_append(const void* k, int64_t k_st, int64_t k_sh, const void* v, int64_t v_st, int64_t v_sh, int dtype,
                                const int32_t* step, int64_t items, int32_t* table, int64_t max_blocks, int64_t H, int64_t D, int64_t P,
                                int code, uint8_t* kc, uint8_t* vc, float* sc, void* ko, void* vo, void* stream) {
  KVQ_PAGES_REQUIRE("kvq_pages_append")
  KVQ_REQUIRE(k && v && step && table && kc && vc && sc && ko && vo, "kvq_pages_append: null pointer");
  KVQ_REQUIRE(reinterpret_cast<uintptr_t>(k) % 16 == 0 && reinterpret_cast<uintptr_t>(v) % 16 == 0 && (k_st | k_sh | v_st | v_sh) % 8 == 0,
              "kvq_pages_append: rows and strides must be multiples of 16 bytes");
  KVQ_REQUIRE(items >= 0 && block_grid(items, H) <= kMaxGrid, "kvq_pages_append: too many blocks");
  if (items == 0) return KVQ_OK;
  const Rows16 kr{static_cast<const uint16_t*>(k), k_st, k_sh}, vr{static_cast<const uint16_t*>(v), v_st, v_sh};
  KVQ_PAGES_DISPATCH(hipLaunchKernelGGL((append_kernel<D_, P_, C_, T_>), dim3(static_cast<uint32_t>(block_grid(items, H))), dim3(kThreads), 0,
                                        static_cast<hipStream_t>(stream), kr, vr, step, table, max_blocks, static_cast<int>(H), kc, vc, sc,
                                        static_cast<uint16_t*>(ko), static_cast<uint16_t*>(vo)))
  KVQ_LAUNCH_CHECK("kvq_pages_append");
  return KVQ_OK;
}

extern "C" int kvq_pages_rows(const int64_t* lens, const uint8_t* open, int64_t slots, const int64_t* seq, int64_t n, const int32_t* table,
                              int64_t max_blocks, int64_t H, int64_t D, int64_t P, int code, int dtype, const uint8_t* kc, const uint8_t* vc,
                              const float* sc, const void* ko, const void* vo, void* k_out, void* v_out, int64_t out_elements, void* stream) {
  KVQ_PAGES_REQUIRE("kvq_pages_rows")
  KVQ_REQUIRE(lens && open && (n == 0 || seq) && table && kc && vc && sc && ko && vo, "kvq_pages_rows: null pointer");
  KVQ_REQUIRE(reinterpret_cast<uintptr_t>(k_out) % 16 == 0 && reinterpret_cast<uintptr_t>(v_out) % 16 == 0,
              "kvq_pages_rows: outputs must be 16-byte aligned");
  int64_t rows = 0, blocks = 0;
  for (int64_t i = 0; i < n; ++i) {
    KVQ_REQUIRE(seq[i] >= 0 && seq[i] < slots, "kvq_pages_rows: no slot %lld (of %lld)", static_cast<long long>(seq[i]),
                static_cast<long long>(slots));
    rows += lens[seq[i]];
    blocks += (lens[seq[i]] + P - 1) / P;
  }
  KVQ_REQUIRE(rows < INT64_C(1) << 31 && block_grid(blocks, H) <= kMaxGrid, "kvq_pages_rows: too many rows");
  KVQ_REQUIRE(out_elements >= rows * H * D && (rows == 0 || (k_out && v_out)), "kvq_pages_rows: outputs of %lld elements, %lld needed",
              static_cast<long long>(out_elements), static_cast<long long>(rows * H * D));
  int64_t row = 0;
  for (int64_t at = 0; at < n; at += kMostWhole) {
    WordBlock w;
    const int64_t m = n - at < kMostWhole ? n - at : kMostWhole;
    int64_t block = 0;
    for (int64_t i = 0; i < m; ++i) {
      const int64_t s = seq[at + i];
      int* e = w.w + kWhole * i;
      e[0] = static_cast<int>(s);
      e[1] = static_cast<int>(lens[s]);
      e[2] = static_cast<int>(row);
      e[3] = static_cast<int>(block);
      e[4] = open[s] & 1;
      row += lens[s];
      block += (lens[s] + P - 1) / P;
    }
    if (block == 0) continue;
    KVQ_PAGES_DISPATCH(hipLaunchKernelGGL((rows_kernel<D_, P_, C_, T_>), dim3(static_cast<uint32_t>(block_grid(block, H))), dim3(kThreads), 0,
                                          static_cast<hipStream_t>(stream), w, static_cast<int>(m), static_cast<int>(block), table, max_blocks, static_cast<int>(H), kc,
                                          vc, sc, static_cast<const uint16_t*>(ko), static_cast<const uint16_t*>(vo),
                                          static_cast<uint16_t*>(k_out), static_cast<uint16_t*>(v_out)))
  }
  KVQ_LAUNCH_CHECK("kvq_pages_rows");
  return KVQ_OK;
}

extern "C" int kvq_pages_fork(int64_t* lens, int32_t* table, int32_t* refs, uint8_t* open, int64_t slots, int64_t max_blocks, int64_t page,
                              const int64_t* src, const int64_t* dst, int64_t n, int64_t layers, int64_t H, int64_t D,
                              int32_t* table_device, void* ko, void* vo, void* stream) {
  KVQ_REQUIRE(lens && table && refs && open && src && dst && (!table_device || (ko && vo)), "kvq_pages_fork: null pointer");
  KVQ_REQUIRE(page_ok(page, D) && H > 0 && layers > 0 && layers * H < 65536, "kvq_pages_fork: bad sizes");
  int64_t bad = -1;
  int64_t i = 0;
  for (; i < n; ++i) {
    if (src[i] < 0 || src[i] >= slots || dst[i] < 0 || dst[i] >= slots || open[dst[i]] & 2 || lens[dst[i]]) { bad = i; break; }
    open[dst[i]] |= 2;                                              // marked as a destination
  }
  int64_t taken = -1;                                               // a destination that is also a source
  for (int64_t m = 0; m < i && bad < 0; ++m)
    if (open[src[m]] & 2) taken = src[m];
  for (int64_t m = 0; m < i; ++m) open[dst[m]] &= 1;
  if (bad >= 0) {
    KVQ_REQUIRE(src[bad] >= 0 && src[bad] < slots && dst[bad] >= 0 && dst[bad] < slots, "kvq_pages_fork: no slot %lld or %lld (of %lld)",
                static_cast<long long>(src[bad]), static_cast<long long>(dst[bad]), static_cast<long long>(slots));
    KVQ_REQUIRE(lens[dst[bad]] == 0, "kvq_pages_fork: slot %lld is in use", static_cast<long long>(dst[bad]));
    KVQ_REQUIRE(false, "kvq_pages_fork: slot %lld is named twice", static_cast<long long>(dst[bad]));
  }
  KVQ_REQUIRE(taken < 0, "kvq_pages_fork: slot %lld is both source and destination", static_cast<long long>(taken));
  for (int64_t at = 0; at < n; at += kWords / 4) {
    ForkPairs f;
    const int64_t m = n - at < kWords / 4 ? n - at : kWords / 4;
    for (int64_t e = 0; e < m; ++e) {
      const int64_t s = src[at + e], d = dst[at + e], blocks = lens[s] / page;
      for (int64_t j = 0; j < blocks; ++j) {
        const int32_t p = table[s * max_blocks + j];
        table[d * max_blocks + j] = p;
        ++refs[p];
      }
      lens[d] = lens[s];
      int* w = f.w + 4 * e;
      w[0] = static_cast<int>(s);
      w[1] = open[s] & 1;
      w[2] = static_cast<int>(d);
      w[3] = static_cast<int>(lens[s]);
      open[d] = 0;
    }
    if (table_device)
      hipLaunchKernelGGL(fork_kernel, dim3(static_cast<uint32_t>(m), static_cast<uint32_t>(layers * H)), dim3(kThreads), 0,
                         static_cast<hipStream_t>(stream), f, table_device, max_blocks, slots, static_cast<int>(H), static_cast<int>(page),
                         static_cast<int>(D), static_cast<uint16_t*>(ko), static_cast<uint16_t*>(vo));
  }
  if (table_device) KVQ_LAUNCH_CHECK("kvq_pages_fork");
  return KVQ_OK;
}

extern "C" int kvq_pages_free(int64_t* lens, const int32_t* table, int32_t* refs, uint8_t* open, int64_t* account, int64_t slots,
                              int64_t max_blocks, int64_t page, const int64_t* seq, int64_t n) {
  KVQ_REQUIRE(lens && table && refs && open && account && (n == 0 || seq), "kvq_pages_free: null pointer");
  for (int64_t i = 0; i < n; ++i)
    KVQ_REQUIRE(seq[i] >= 0 && seq[i] < slots, "kvq_pages_free: no slot %lld (of %lld)", static_cast<long long>(seq[i]),
                static_cast<long long>(slots));
  for (int64_t i = 0; i < n; ++i) {
    const int64_t s = seq[i];
    for (int64_t j = 0; j < lens[s] / page; ++j) {
      const int32_t p = table[s * max_blocks + j];
      if (--refs[p] == 0) {
        ++account[0];
        if (p < account[1]) account[1] = p;
      }
    }
    lens[s] = 0;
    open[s] = 0;
  }
  return KVQ_OK;
}

extern "C" int kvq_pages_move(const int64_t* lens, int32_t* table, const int32_t* refs, int32_t* refs_to, int64_t* account, int64_t slots,
                              int64_t pages, int64_t pages_to, int64_t end, int64_t max_blocks, int64_t page, int32_t* place, int64_t layers,
                              int64_t H, int64_t D, const uint8_t* kc, const uint8_t* vc, const float* sc, uint8_t* kc_to, uint8_t* vc_to,
                              float* sc_to, int32_t* table_device, void* stream) {
  KVQ_REQUIRE(lens && table && refs && refs_to && account && place, "kvq_pages_move: null pointer");
  KVQ_REQUIRE(page_ok(page, D) && H > 0 && layers > 0 && layers < 65536 && pages < INT64_C(1) << 31 && pages_to < INT64_C(1) << 31 &&
                  end >= 0 && end <= pages_to,
              "kvq_pages_move: bad sizes");
  KVQ_REQUIRE(!table_device || (kc && vc && sc && kc_to && vc_to && sc_to), "kvq_pages_move: null pointer");
  const bool same = refs == refs_to;          // the pools may be null where only the accounts move
  KVQ_REQUIRE((!same || pages == pages_to) && (!table_device || same == (kc == kc_to)), "kvq_pages_move: one pool has one size");
  int64_t used = 0;
  for (int64_t p = 0; p < pages; ++p) used += refs[p] != 0;
  KVQ_REQUIRE(used <= end, "kvq_pages_move: %lld pages are in use", static_cast<long long>(used));
  // pages from `end` on to the lowest free places, in order
  int64_t hole = 0;
  for (int64_t p = 0; p < pages; ++p) {
    place[p] = static_cast<int32_t>(p);
    if (refs[p] && p >= end) {
      while (hole < pages && refs[hole]) ++hole;
      place[p] = static_cast<int32_t>(hole++);
    }
  }
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (table_device) {
    const Pool s{const_cast<uint8_t*>(kc), const_cast<uint8_t*>(vc), const_cast<float*>(sc)}, d{kc_to, vc_to, sc_to};
    Moves m;
    int n = 0;
    auto flush = [&] {
      if (n) hipLaunchKernelGGL(move_kernel, dim3(n, static_cast<uint32_t>(layers)), dim3(kThreads), 0, st, m, s, d, pages, pages_to,
                                static_cast<int>(H), H * D * page);
      n = 0;
    };
    for (int64_t p = 0; p < pages; ++p) {
      if (!refs[p] || (same && place[p] == p)) continue;
      m.w[2 * n] = static_cast<int>(p);
      m.w[2 * n + 1] = place[p];
      if (++n == kWords / 2) flush();
    }
    flush();
    if (pages_to < pages) {
      const int64_t entries = slots * max_blocks;
      KVQ_REQUIRE(entries / kThreads < kMaxGrid, "kvq_pages_move: the table is too large");
      hipLaunchKernelGGL(clip_kernel, dim3(static_cast<uint32_t>((entries + kThreads - 1) / kThreads)), dim3(kThreads), 0, st, table_device,
                         entries, static_cast<int>(pages_to));
    }
  }
  Patches c;
  int n = 0;
  auto flush = [&] {
    if (n && table_device) hipLaunchKernelGGL(patch_kernel, dim3(1), dim3(kThreads), 0, st, c, n, table_device, max_blocks);
    n = 0;
  };
  for (int64_t i = 0; i < slots; ++i)
    for (int64_t j = 0; j < lens[i] / page; ++j) {
      int32_t& p = table[i * max_blocks + j];
      if (place[p] == p) continue;
      p = place[p];
      c.w[3 * n] = static_cast<int>(i);
      c.w[3 * n + 1] = static_cast<int>(j);
      c.w[3 * n + 2] = p;
      if (++n == kWords / 3) flush();
    }
  flush();
  if (!same) memset(refs_to, 0, sizeof(int32_t) * pages_to);
  for (int64_t p = 0; p < pages; ++p) {
    if (!refs[p] || (same && place[p] == p)) continue;
    refs_to[place[p]] = refs[p];                                    // in place: to a page that was free
    if (same) refs_to[p] = 0;
  }
  account[0] = pages_to - used;
  account[1] = 0;
  if (table_device) KVQ_LAUNCH_CHECK("kvq_pages_move");
  return KVQ_OK;
}
