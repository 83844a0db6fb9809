// Attention over whole prompts: packed sequences of any lengths, grouped heads, causal with the last
// query at the last key (a chunk of a prompt behind its past) or over all keys.
//
// A workgroup takes 128 rows of one KV head: (token, query head) pairs, token major, so that the query
// heads of a group share the keys and values that are staged in LDS, 64 tokens at a time.  Each of its
// four wavefronts holds 32 rows as the columns of the matrix products: S^T = K Q^T, the softmax in base
// 2 with one running maximum and sum per column (two lanes hold a column; one swap joins them), and
// O^T += V^T P^T.  The accumulator layout of S^T is the operand layout of P^T once V^T takes its tokens in
// the same order, so probabilities never leave their lanes: V^T comes from LDS by transposing reads.
// Probabilities are rounded to the inputs' type (half a step of the output's type); the sums, the
// maximum and the accumulators are float32.
#include <algorithm>
#include <type_traits>

#include "mfma_common.hpp"

namespace kvq {
namespace {

constexpr int kThreads = 256, kTileRows = 128, kTileKeys = 64, kItemWords = 8;

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;

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

struct PromptArgs {
  const uint16_t *q, *k, *v;
  int64_t q_st, q_sh, k_st, k_sh, v_st, v_sh;
  const int* items;                           // {first row, tokens, first key, keys, visible to the first token, step}
  int H, rep;
  float scale;                                // scaling * log2(e)
  uint16_t* out;                              // (rows, Hq, D)
};

template <int D, bool BF16>
__global__ __launch_bounds__(kThreads, 2) void prompt_kernel(PromptArgs a) {
  constexpr int kRow = D / 8, kPer = kTileKeys * kRow / kThreads;   // 16-byte pieces of a row, of a thread
  constexpr int kKMask = kRow - 1, kVMask = kRow / 2 - 1;
  constexpr uint32_t kInf = BF16 ? 0x7f80u : 0x7c00u;
  __shared__ __align__(16) uint16_t ks[kTileKeys * D], vs[kTileKeys * D];
  __shared__ int flag;
  const int* it = a.items + kItemWords * (blockIdx.x / a.H);
  const int h = blockIdx.x % a.H;
  const int row0 = it[0], toks = it[1], key0 = it[2], keys = it[3], vis0 = it[4], vis_step = it[5];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, col = lane & 31, g = lane >> 5;

  const int row = wave * 32 + col, tok = row / a.rep, hq = row % a.rep;
  const bool live = tok < toks;
  int visible = vis0 + vis_step * tok;
  visible = !live ? 0 : visible < keys ? visible : keys;
  u32x4 q[D / 16];
  {
    const uint16_t* qp = a.q + (row0 + static_cast<int64_t>(live ? tok : 0)) * a.q_st + (static_cast<int64_t>(h) * a.rep + hq) * a.q_sh + 8 * g;
#pragma unroll
    for (int i = 0; i < D / 16; ++i) {
      const uint4 x = *reinterpret_cast<const uint4*>(qp + 16 * i);
      q[i] = live ? u32x4{x.x, x.y, x.z, x.w} : u32x4{0, 0, 0, 0};
    }
  }
  f32x16 o[D / 32];
#pragma unroll
  for (int c = 0; c < D / 32; ++c)
#pragma unroll
    for (int e = 0; e < 16; ++e) o[c][e] = 0.0f;
  float m = -INFINITY, l = 0.0f;

  const uint16_t* kb = a.k + static_cast<int64_t>(key0) * a.k_st + h * a.k_sh;
  const uint16_t* vb = a.v + static_cast<int64_t>(key0) * a.v_st + h * a.v_sh;
  uint4 kr[kPer], vr[kPer];
  auto load = [&](int j) {                    // keys behind the last one: the last one again (masked)
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int p = tid + i * kThreads, c = p % kRow * 8;
      int64_t r = j * kTileKeys + p / kRow;
      r = r < keys ? r : keys - 1;
      kr[i] = *reinterpret_cast<const uint4*>(kb + r * a.k_st + c);
      vr[i] = *reinterpret_cast<const uint4*>(vb + r * a.v_st + c);
    }
  };
  const int tiles = (keys + kTileKeys - 1) / kTileKeys;
  // tiles that every row sees whole
  int open = vis0 < keys ? vis0 : keys;
  open = open < 0 ? 0 : open / kTileKeys;
  if (tid == 0) flag = 0;
  if (tiles > 0) load(0);

  for (int j = 0; j < tiles; ++j) {
    const bool masked = j >= open;
    __syncthreads();
    if (masked) {
      // a value that is hidden from some row may be an infinity or a NaN
      bool bad = false;
#pragma unroll
      for (int i = 0; i < kPer; ++i) {
        const uint32_t w[4] = {vr[i].x, vr[i].y, vr[i].z, vr[i].w};
#pragma unroll
        for (int e = 0; e < 4; ++e) bad |= (w[e] & kInf) == kInf || (w[e] >> 16 & kInf) == kInf;
      }
      if (bad) flag = j + 1;
    }
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int p = tid + i * kThreads, r = p / kRow, c = p % kRow;
      *reinterpret_cast<uint4*>(ks + r * D + (c ^ (r & kKMask)) * 8) = kr[i];
      *reinterpret_cast<uint4*>(vs + r * D + (c ^ ((r & kVMask) << 1)) * 8) = vr[i];
    }
    __syncthreads();
    const bool bad = masked && flag == j + 1;
    if (j + 1 < tiles) load(j + 1);

    float t[32];
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      f32x16 s;
#pragma unroll
      for (int e = 0; e < 16; ++e) s[e] = 0.0f;
#pragma unroll
      for (int i = 0; i < D / 16; ++i) {
        const uint4 w = *reinterpret_cast<const uint4*>(ks + (32 * x + col) * D + ((2 * i + g) ^ (col & kKMask)) * 8);
        s = mfma32<BF16>(u32x4{w.x, w.y, w.z, w.w}, q[i], s);
      }
#pragma unroll
      for (int e = 0; e < 16; ++e) t[16 * x + e] = s[e] * a.scale;
    }
    // register 16 x + 4 b + e of lane half g: token 32 x + 8 b + 4 g + e
    if (masked) {
      const int lim = visible - j * kTileKeys - 4 * g;
#pragma unroll
      for (int i = 0; i < 32; ++i) t[i] = 32 * (i / 16) + 8 * (i / 4 % 4) + i % 4 < lim ? t[i] : -INFINITY;
    }
    float top = t[0];
#pragma unroll
    for (int i = 1; i < 32; ++i) top = fmaxf(top, t[i]);
    top = fmaxf(m, xmax32(top));
    const float safe = top == -INFINITY ? 0.0f : top, old = __builtin_amdgcn_exp2f(m - safe);
    float sum = 0.0f;
#pragma unroll
    for (int i = 0; i < 32; ++i) {
      t[i] = __builtin_amdgcn_exp2f(t[i] - safe);
      sum += t[i];
    }
    l = l * old + sum;
    m = top;
    if (__builtin_amdgcn_ballot_w64(old != 1.0f)) {
#pragma unroll
      for (int c = 0; c < D / 32; ++c) o[c] *= old;
    }
    // 16 tokens a product; this lane's: 16 y + 4 g + e and 16 y + 8 + 4 g + e
    const int tr = (lane & 15) >> 2, tc = (lane >> 4 & 1) * 16 + (lane & 3) * 4;
#pragma unroll
    for (int y = 0; y < 4; ++y) {
      u32x4 p;
#pragma unroll
      for (int e = 0; e < 4; ++e) p[e] = pack2<BF16>(t[8 * y + 2 * e], t[8 * y + 2 * e + 1]);
#pragma unroll
      for (int c = 0; c < D / 32; ++c) {
        u32x4 w;
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int r = 16 * y + 8 * e + 4 * g + tr, ch = 32 * c + tc;
          const u32x2 z = read_tr(vs + r * D + ((ch / 8) ^ ((r & kVMask) << 1)) * 8 + ch % 8);
          w[2 * e] = z[0];
          w[2 * e + 1] = z[1];
        }
        if (bad) {
#pragma unroll
          for (int e = 0; e < 4; ++e)
            w[e] = ((w[e] & kInf) == kInf ? 0u : w[e] & 0xffffu) | ((w[e] >> 16 & kInf) == kInf ? 0u : w[e] & 0xffff0000u);
        }
        o[c] = mfma32<BF16>(w, p, o[c]);
      }
    }
    if (bad) {                                // the rows that do see such a value get it
      for (int r = 0; r < kTileKeys; ++r) {
        const bool sees = j * kTileKeys + r < visible;
#pragma unroll
        for (int c = 0; c < D / 32; ++c)
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            const int ch = 32 * c + 8 * (e / 4) + 4 * g + e % 4;
            const uint16_t x = vs[r * D + ((ch / 8) ^ ((r & kVMask) << 1)) * 8 + ch % 8];
            if (sees && (x & kInf) == kInf) o[c][e] += BF16 ? bf16_to_f32(x) : f16_to_f32(x);
          }
      }
    }
  }

  if (!live) return;
  l = xsum32(l);
  const float inv = visible > 0 ? 1.0f / l : 0.0f;                  // a row without a visible key: zeros
  uint16_t* out = a.out + ((row0 + static_cast<int64_t>(tok)) * a.H * a.rep + h * a.rep + hq) * D + 4 * g;
#pragma unroll
  for (int c = 0; c < D / 32; ++c)
#pragma unroll
    for (int e = 0; e < 4; ++e)
      *reinterpret_cast<uint2*>(out + 32 * c + 8 * e) = make_uint2(pack2<BF16>(o[c][4 * e] * inv, o[c][4 * e + 1] * inv),
                                                                   pack2<BF16>(o[c][4 * e + 2] * inv, o[c][4 * e + 3] * inv));
}

struct Item {
  int32_t w[kItemWords];
};

}  // namespace
}  // namespace kvq

using namespace kvq;

extern "C" int64_t kvq_prompt_plan(const int64_t* lens_q, const int64_t* lens_k, int64_t n, int64_t rep, int causal, int32_t* items,
                                   int64_t items_cap) {
  if (n < 0 || (n && (!lens_q || !lens_k)) || rep < 1 || rep > kTileRows) return -1;
  const int64_t per = kTileRows / rep;        // tokens of a tile
  int64_t total = 0, row = 0, key = 0;
  Item* out = reinterpret_cast<Item*>(items);
  for (int64_t i = 0; i < n; ++i) {
    const int64_t lq = lens_q[i], lk = lens_k[i];
    if (lq < 0 || lk < 0 || lq >= INT64_C(1) << 31 || lk >= INT64_C(1) << 31) return -1;
    for (int64_t t = 0; t < lq; t += per, ++total) {
      if (!items || total >= items_cap) continue;
      const int64_t toks = lq - t < per ? lq - t : per, vis0 = causal ? lk - lq + t + 1 : lk;
      int64_t keys = causal ? vis0 + toks - 1 : lk;
      keys = keys < 0 ? 0 : keys;
      out[total] = {static_cast<int32_t>(row + t), static_cast<int32_t>(toks), static_cast<int32_t>(key), static_cast<int32_t>(keys),
                    static_cast<int32_t>(vis0), causal ? 1 : 0, 0, 0};
    }
    row += lq;
    key += lk;
    if (row >= INT64_C(1) << 31 || key >= INT64_C(1) << 31) return -1;
  }
  // the longest first: the last workgroups to end are short ones
  if (items && total <= items_cap)
    std::sort(out, out + total, [](const Item& x, const Item& y) { return x.w[3] != y.w[3] ? x.w[3] > y.w[3] : x.w[0] < y.w[0]; });
  return total;
}

extern "C" int kvq_prompt_attention(const void* q, int64_t q_st, int64_t q_sh, const void* k, int64_t k_st, int64_t k_sh, const void* v,
                                    int64_t v_st, int64_t v_sh, int dtype, int64_t Hq, int64_t H, int64_t D, float scaling,
                                    const int32_t* items, int64_t n_items, void* out, void* stream) {
  KVQ_REQUIRE(D == 64 || D == 128, "kvq_prompt_attention: head_dim must be 64 or 128 (got %lld)", static_cast<long long>(D));
  KVQ_REQUIRE(dtype == KVQ_F16 || dtype == KVQ_BF16, "kvq_prompt_attention: rows must be fp16 or bf16");
  KVQ_REQUIRE(H > 0 && Hq > 0 && Hq % H == 0 && Hq / H <= kTileRows && n_items >= 0, "kvq_prompt_attention: bad sizes");
  if (n_items == 0) return KVQ_OK;
  KVQ_REQUIRE(q && k && v && items && out, "kvq_prompt_attention: null pointer");
  KVQ_REQUIRE((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v) |
               reinterpret_cast<uintptr_t>(out)) % 16 == 0 && (q_st | q_sh | k_st | k_sh | v_st | v_sh) % 8 == 0,
              "kvq_prompt_attention: rows and strides must be multiples of 16 bytes");
  KVQ_REQUIRE(n_items * H < INT64_C(1) << 31, "kvq_prompt_attention: too many rows");
  const PromptArgs a{static_cast<const uint16_t*>(q), static_cast<const uint16_t*>(k), static_cast<const uint16_t*>(v),
                     q_st, q_sh, k_st, k_sh, v_st, v_sh, items, static_cast<int>(H), static_cast<int>(Hq / H),
                     scaling * 1.44269504088896341f, static_cast<uint16_t*>(out)};
  const dim3 grid(static_cast<uint32_t>(n_items * H));
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (D == 128 && dtype == KVQ_BF16) hipLaunchKernelGGL((prompt_kernel<128, true>), grid, dim3(kThreads), 0, s, a);
  else if (D == 128) hipLaunchKernelGGL((prompt_kernel<128, false>), grid, dim3(kThreads), 0, s, a);
  else if (dtype == KVQ_BF16) hipLaunchKernelGGL((prompt_kernel<64, true>), grid, dim3(kThreads), 0, s, a);
  else hipLaunchKernelGGL((prompt_kernel<64, false>), grid, dim3(kThreads), 0, s, a);
  KVQ_LAUNCH_CHECK("kvq_prompt_attention");
  return KVQ_OK;
}
