// The paged cache's accounts in device memory: page tables, slot maps and a step's description (pages.hpp) from the
// lengths that requests have there, and pages given back, without the host.
//
// A step of n sequences takes counts[i] of at most `most` tokens, known on the device only; its rows lie at i * most.
// extend: one workgroup checks the counts, finds the lowest free pages, cuts the decode's work and writes the sequences' and
// runs' entries (scans over the sequences, 1024 at a time), and what is there per page and per row, or a second launch does where
// that is much.
// A step that does not fit changes no slot and is counted: it describes no tokens.
// What bounds them: round trips of a single workgroup; the whole of it is a few KB.  extend for 8 sequences of one token 3.9-5 us, of
// up to 900 tokens 8-9; for 256 sequences of four tokens 8.7, of up to 700 8.9 and 2-4 for the second
// launch; free 3.5 for 8 sequences, 5 for 256.
#include <type_traits>

#include "pages.hpp"

namespace kvq {
namespace {

constexpr int kMostThreads = 1024, kRowThreads = 256, kFound = 4096;

struct Tables {
  const int *slots, *counts;                  // of the step's sequences
  int n, most, P, shift, max_tokens;          // P = 1 << shift
  int64_t pages, max_blocks;
  int splits;                                 // split items at most
  int *lens, *refs, *open;                    // (slots), (pages), (slots)
  int* account;                               // {free pages, no free page below this one, steps refused}
  int* table;
  int* desc;
  int *found, *rank;                          // the step's new pages in order; each sequence's first of them
  int* positions;                             // (n most) or none: of each row in its sequence, -1 for none
  int64_t* places;                            // (n most): page * P + offset of a row whose block is full, else -1
};

__device__ __forceinline__ int units_of(int len, int shift) {
  const int full = len >> shift << shift;
  return (full + kUnit - 1) / kUnit + (len - full + kUnit - 1) / kUnit;
}

typedef int i32x4 __attribute__((ext_vector_type(4)));

__device__ __forceinline__ int wave_total(int x) {
#pragma unroll
  for (int o = 32; o; o >>= 1) x += __shfl_xor(x, o);
  return x;
}

// Four sums of the lower threads of a workgroup of W wavefronts, N of them used; `total` of all threads
template <int N, int W>
__device__ __forceinline__ i32x4 scan(i32x4 x, i32x4& total, i32x4 (&room)[W]) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  i32x4 sum = x;
#pragma unroll
  for (int k = 0; k < N; ++k)
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const int y = __shfl_up(sum[k], o);
      sum[k] += lane >= o ? y : 0;
    }
  if (lane == 63) room[wave] = sum;
  __syncthreads();
  i32x4 before = {0, 0, 0, 0}, all = {0, 0, 0, 0};
#pragma unroll
  for (int w = 0; w < W; ++w) {
    const i32x4 y = room[w];
    if (w < wave) before += y;
    all += y;
  }
  total = all;
  __syncthreads();                            // the room is free again
  return sum - x + before;
}

// T threads; WHOLE: at most T sequences, with their pages and rows written in this launch
template <int T, bool WHOLE>
__global__ __launch_bounds__(T) void tables_extend_kernel(Tables a) {
  constexpr int kWaves = T / 64, kTries = 16, kLook = 8;    // pages a thread looks at at once
  __shared__ i32x4 room[kWaves];
  __shared__ int units[T], tops[kWaves][2], fits[kTries], flags, last_page;
  __shared__ int found_here[WHOLE ? kFound : 1], pos[WHOLE ? T : 1], count[WHOLE ? T : 1], ranks[WHOLE ? T : 1], item0[WHOLE ? T : 1];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  int* found = WHOLE ? found_here : a.found;
  if (tid == 0) flags = 0;

  // what the step needs, and whether it may have it; the first T sequences stay in registers
  int need = 0, all = 0, active = 0, longest = 0, most_units = 4, bad = 0;
  int own_s = 0, own_c = 0, own_pos = 0, own_open = 0;
  for (int i = tid; i < a.n; i += T) {
    const int s = a.slots[i], c = a.counts[i], pos0 = a.lens[s], open = a.open[s];
    const bool ok = c >= 0 && c <= a.most && static_cast<int64_t>(pos0) + c <= a.max_tokens;
    bad |= !ok;
    const int end = ok ? pos0 + c : pos0, u = ok && c ? units_of(end, a.shift) : 0;
    need += (end >> a.shift) - (pos0 >> a.shift);
    all += u;
    active += ok && c;
    longest = ok && c > longest ? c : longest;
    most_units = u > most_units ? u : most_units;
    if (i < T) {
      units[i] = u;
      own_s = s;
      own_c = c;
      own_pos = pos0;
      own_open = open;
    }
  }
  const int free_pages = a.account[0], low = a.account[1];
  need = wave_total(need);
  all = wave_total(all);
  active = wave_total(active);
  bad = wave_total(bad);
#pragma unroll
  for (int o = 32; o; o >>= 1) {
    const int x = __shfl_xor(longest, o), y = __shfl_xor(most_units, o);
    longest = x > longest ? x : longest;
    most_units = y > most_units ? y : most_units;
  }
  if (lane == 0) {
    room[wave] = i32x4{need, all, active, bad};
    tops[wave][0] = longest;
    tops[wave][1] = most_units;
  }
  __syncthreads();
  i32x4 total = {0, 0, 0, 0};
#pragma unroll
  for (int w = 0; w < kWaves; ++w) {
    total += room[w];
    longest = tops[w][0] > longest ? tops[w][0] : longest;
    most_units = tops[w][1] > most_units ? tops[w][1] : most_units;
  }
  __syncthreads();                            // the room is free for the scans
  const bool fit = !total[3] && total[0] <= free_pages;
  need = fit ? total[0] : 0;
  all = fit ? total[1] : 0;
  active = fit ? total[2] : 0;
  longest = fit ? longest : 0;

  // Units of a split item: few enough that there are a.splits items at most.  With u units in all and k sequences, u /
  // (splits - k) are; of 16 sizes down to an even share the smallest that fits is taken, T / 16 threads for each.
  int per = most_units;
  if (a.splits > active) {
    const int safe = (all - 1) / (a.splits - active) + 1;
    per = safe < 4 ? 4 : safe < most_units ? safe : most_units;
  }
  const int share = (all - 1) / a.splits + 1, least = share < 4 ? 4 : share < per ? share : per;
  if (a.n <= T && least < per) {
    constexpr int kEach = T / kTries;
    const int mine = least + static_cast<int>(static_cast<int64_t>(per - least) * (tid / kEach) / kTries);
    int items = 0;
    for (int i = tid % kEach; i < a.n; i += kEach) items += (units[i] + mine - 1) / mine;
#pragma unroll
    for (int o = kEach / 2; o; o >>= 1) items += __shfl_xor(items, o);
    if (tid % kEach == 0) fits[tid / kEach] = items <= a.splits ? mine : per;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kTries; ++w) per = fits[w] < per ? fits[w] : per;
  }

  // the lowest free pages, in order
  int got = 0;
  for (int64_t at = low; got < need && at < a.pages; at += kLook * T) {
    const int64_t p = at + kLook * tid;
    bool is[kLook];
    i32x4 free_here = {0, 0, 0, 0};
#pragma unroll
    for (int k = 0; k < kLook; ++k) {
      is[k] = p + k < a.pages && a.refs[p + k < a.pages ? p + k : a.pages - 1] == 0;
      free_here[0] += is[k];
    }
    int rank = got + scan<1, kWaves>(free_here, total, room)[0];
#pragma unroll
    for (int k = 0; k < kLook; ++k) {
      if (!is[k]) continue;
      if (rank < need) {
        found[rank] = static_cast<int>(p + k);
        a.refs[p + k] = 1;
        if (rank == need - 1) last_page = static_cast<int>(p + k);
      }
      ++rank;
    }
    got += total[0];
  }

  // entries of the sequences and their runs
  int* seqs = a.desc + kStepHead;
  int* runs = seqs + kStepSeq * (a.n + 1);
  const int pages_at = kStepHead + kStepSeq * (a.n + 1) + kStepRun * (2 * a.n + 1);
  i32x4 carry = {0, 0, 0, 0};                 // pages, items, split items, tokens of these
  int odd = 0;                                // 1: not an item each, 2: not a split item each, 4: several of one
  for (int i0 = 0; i0 < a.n; i0 += T) {
    const int i = i0 + tid;
    const bool in = i < a.n, own = WHOLE || i0 == 0;
    const int s = own ? own_s : in ? a.slots[i] : 0, c = !in || !fit ? 0 : own ? own_c : a.counts[i], pos0 = own ? own_pos : in ? a.lens[s] : 0;
    const int end = pos0 + c, src = (own ? own_open : in ? a.open[s] : 0) & 1;
    const int dst = (pos0 & (a.P - 1)) && (end >> a.shift) > (pos0 >> a.shift) && (end & (a.P - 1)) ? src ^ 1 : src;
    const int u = c ? units_of(end, a.shift) : 0, items = c ? ((end - 1) >> a.shift) - (pos0 >> a.shift) + 1 : 0, split = (u + per - 1) / per;
    if (in) odd |= (items != 1) | (split != 1) << 1 | (split > 1) << 2;
    if (i0 + T >= a.n && odd) atomicOr(&flags, odd);
    const i32x4 x = carry + scan<4, kWaves>(i32x4{(end >> a.shift) - (pos0 >> a.shift), items, split, split * c}, total, room);
    if (in) {
      int* e = seqs + kStepSeq * i;
      e[0] = s;
      e[1] = pos0;
      e[2] = c;
      e[3] = i * a.most;
      e[4] = x[1];
      e[5] = i;
      e[6] = src | dst << 1;
      e[7] = 0;
      int* r = runs + kStepRun * i;
      r[0] = s;
      r[1] = i * a.most;
      r[2] = c;
      r[3] = 0;
      r[4] = u;
      r[5] = x[2];
      r[6] = x[3];
      r[7] = i;
      r[8] = pos0;
      r[9] = dst;
      r[10] = 0;
      r[11] = split;
      if constexpr (WHOLE) {
        pos[i] = pos0;
        count[i] = c;
        ranks[i] = x[0];
        item0[i] = x[1];
        units[i] = s;                         // from here on
      } else {
        a.rank[i] = x[0];
      }
      if (c) {
        a.lens[s] = end;
        a.open[s] = dst;
      }
    }
    carry += total;
  }
  if (tid == 0) {
    int* e = seqs + kStepSeq * a.n;
    for (int k = 0; k < kStepSeq; ++k) e[k] = 0;
    e[3] = a.n * a.most;
    e[4] = carry[1];
    e[5] = a.n;
    int* r = runs + kStepRun * a.n;
    for (int k = 0; k < kStepRun; ++k) r[k] = 0;
    r[5] = carry[2];
    r[6] = carry[3];
    int* d = a.desc;
    d[0] = a.n;
    d[1] = carry[1];
    d[2] = carry[2];
    d[3] = per;
    d[4] = !(flags & 1);
    d[5] = longest;
    d[6] = longest;
    d[7] = carry[3];
    d[8] = a.n;
    d[9] = pages_at;
    d[10] = flags >> 2 & 1;
    d[11] = !(flags & 2);
    a.account[0] = free_pages - need;
    if (need) a.account[1] = last_page + 1;
    if (!fit) a.account[2] += 1;
  }
  if constexpr (WHOLE) {
    __syncthreads();
    const int most_items = ((a.most + a.P - 2) >> a.shift) + 1;
    for (int at = tid; at < a.n * most_items; at += T) {
      const int i = at / most_items, j = at % most_items, first = (pos[i] >> a.shift), end = pos[i] + count[i];
      if (!count[i] || j > ((end - 1) >> a.shift) - first) continue;
      const int page = j < (end >> a.shift) - first ? found[ranks[i] + j] : -1;
      a.desc[pages_at + item0[i] + j] = page;
      if (page >= 0) a.table[units[i] * a.max_blocks + first + j] = page;
    }
    for (int row = tid; row < a.n * a.most; row += T) {
      const int i = row / a.most, j = row % a.most, first = (pos[i] >> a.shift), at = pos[i] + j, block = (at >> a.shift) - first;
      const bool in = j < count[i];
      a.positions[row] = in ? at : -1;
      a.places[row] = in && block < ((pos[i] + count[i]) >> a.shift) - first ? static_cast<int64_t>(found[ranks[i] + block]) * a.P + (at & (a.P - 1)) : -1;
    }
  }
}

// Workgroup (sequence, piece of its rows): the table's new entries, the items' pages, positions and places
__global__ __launch_bounds__(kRowThreads) void tables_rows_kernel(Tables a) {
  const StepSeq s = step_seq(a.desc, blockIdx.x);
  const int rank = a.rank[blockIdx.x], first = (s.pos0 >> a.shift), end = s.pos0 + s.count, new_pages = (end >> a.shift) - first;
  const int items = s.count ? ((end - 1) >> a.shift) - first + 1 : 0;
  const int stride = kRowThreads * gridDim.y, at = blockIdx.y * kRowThreads + threadIdx.x;
  int* item_page = a.desc + a.desc[9] + s.item0;
  for (int j = at; j < items; j += stride) {
    const int page = j < new_pages ? a.found[rank + j] : -1;
    item_page[j] = page;
    if (page >= 0) a.table[s.slot * a.max_blocks + first + j] = page;
  }
  for (int j = at; j < a.most; j += stride) {
    const int64_t row = static_cast<int64_t>(blockIdx.x) * a.most + j;
    const int pos = s.pos0 + j, block = (pos >> a.shift) - first;
    const bool in = j < s.count;
    a.positions[row] = in ? pos : -1;
    a.places[row] = in && block < new_pages ? static_cast<int64_t>(a.found[rank + block]) * a.P + (pos & (a.P - 1)) : -1;
  }
}

// Workgroup per sequence: its pages' counts, one less
__global__ __launch_bounds__(kRowThreads) void tables_free_kernel(Tables a, const uint8_t* __restrict__ which) {
  __shared__ int sums[2];
  if (which && !which[blockIdx.x]) return;
  const int s = a.slots[blockIdx.x], blocks = (a.lens[s] >> a.shift);
  if (threadIdx.x == 0) {
    sums[0] = 0;
    sums[1] = 0x7fffffff;
  }
  __syncthreads();                            // and everyone has the length
  int freed = 0, low = 0x7fffffff;
  for (int j = threadIdx.x; j < blocks; j += kRowThreads) {
    const int page = a.table[s * a.max_blocks + j];
    if (atomicSub(a.refs + page, 1) != 1) continue;
    ++freed;
    low = page < low ? page : low;
  }
  if (freed) {
    atomicAdd(sums, freed);
    atomicMin(sums + 1, low);
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    a.lens[s] = 0;
    a.open[s] = 0;
    if (sums[0]) {
      atomicAdd(a.account, sums[0]);
      atomicMin(a.account + 1, sums[1]);
    }
  }
}

}  // namespace
}  // namespace kvq

using namespace kvq;

extern "C" int64_t kvq_tables_step_words(int64_t page, int64_t n, int64_t most) {
  if (n < 1 || most < 1 || n >= INT64_C(1) << 31 || most >= INT64_C(1) << 31 || n * most >= INT64_C(1) << 31 || (page != 32 && page != 64 && page != 128)) return -1;
  const int64_t items = n * ((most + page - 2) / page + 1), words = kStepHead + kStepSeq * (n + 1) + kStepRun * (2 * n + 1) + items;
  return words < INT64_C(1) << 31 ? words : -1;
}

extern "C" int kvq_tables_extend(const int32_t* slots, const int32_t* counts, int64_t n, int64_t most, int64_t page, int64_t max_tokens,
                                 int64_t pages, int64_t max_blocks, int64_t splits, int32_t* lens, int32_t* refs, int32_t* open,
                                 int32_t* account, int32_t* table, int32_t* desc, int64_t desc_words, int32_t* scratch,
                                 int64_t scratch_words, int32_t* positions, int64_t* places, void* stream) {
  const int64_t words = kvq_tables_step_words(page, n, most);
  KVQ_REQUIRE(words >= 0, "kvq_tables_extend: bad sizes");
  KVQ_REQUIRE(slots && counts && lens && refs && open && account && table && desc && scratch && positions && places,
              "kvq_tables_extend: null pointer");
  const int64_t items = words - kStepHead - kStepSeq * (n + 1) - kStepRun * (2 * n + 1);
  KVQ_REQUIRE(desc_words >= words && scratch_words >= n + items, "kvq_tables_extend: a short description or scratch");
  KVQ_REQUIRE(max_tokens > 0 && max_tokens < INT64_C(1) << 31 && pages > 0 && pages < INT64_C(1) << 31 && max_blocks >= (max_tokens + page - 1) / page &&
                  n <= (INT64_C(1) << 29) / ((max_tokens + 31) / 32),  // all sums stay below 2^31
              "kvq_tables_extend: bad sizes");
  KVQ_REQUIRE(splits >= n && splits * most < INT64_C(1) << 31, "kvq_tables_extend: at least one split item per sequence is needed, and below 2^31 tokens of them");
  const Tables a{slots, counts, static_cast<int>(n), static_cast<int>(most), static_cast<int>(page), __builtin_ctz(static_cast<unsigned>(page)), static_cast<int>(max_tokens), pages, max_blocks,
                 static_cast<int>(splits), lens, refs, open, account, table, desc, scratch + n, scratch, positions, places};
  hipStream_t s = static_cast<hipStream_t>(stream);
  // in one launch where a workgroup holds the sequences and the pages: 8 sequences with their prompts 15 us in two, 8 in one
  if (n <= kMostThreads && items <= kFound && n * most <= 16384) {
    if (n <= 256) hipLaunchKernelGGL((tables_extend_kernel<256, true>), dim3(1), dim3(256), 0, s, a);
    else hipLaunchKernelGGL((tables_extend_kernel<kMostThreads, true>), dim3(1), dim3(kMostThreads), 0, s, a);
    KVQ_LAUNCH_CHECK("kvq_tables_extend");
    return KVQ_OK;
  }
  const uint32_t pieces = static_cast<uint32_t>((most + 16 * kRowThreads - 1) / (16 * kRowThreads));
  KVQ_REQUIRE(n * pieces <= kMaxGrid && pieces < 65536, "kvq_tables_extend: too many rows");
  if (n <= 256) hipLaunchKernelGGL((tables_extend_kernel<256, false>), dim3(1), dim3(256), 0, s, a);
  else hipLaunchKernelGGL((tables_extend_kernel<kMostThreads, false>), dim3(1), dim3(kMostThreads), 0, s, a);
  hipLaunchKernelGGL(tables_rows_kernel, dim3(static_cast<uint32_t>(n), pieces), dim3(kRowThreads), 0, s, a);
  KVQ_LAUNCH_CHECK("kvq_tables_extend");
  return KVQ_OK;
}

extern "C" int kvq_tables_free(const int32_t* slots, const uint8_t* which, int64_t n, int64_t page, int64_t max_blocks, int32_t* lens,
                               int32_t* refs, int32_t* open, int32_t* account, const int32_t* table, void* stream) {
  KVQ_REQUIRE(n >= 1 && n <= kMaxGrid && (page == 32 || page == 64 || page == 128) && max_blocks >= 1, "kvq_tables_free: bad sizes");
  KVQ_REQUIRE(slots && lens && refs && open && account && table, "kvq_tables_free: null pointer");
  Tables a{};
  a.slots = slots;
  a.n = static_cast<int>(n);
  a.P = static_cast<int>(page);
  a.shift = __builtin_ctz(static_cast<unsigned>(page));
  a.max_blocks = max_blocks;
  a.lens = lens;
  a.refs = refs;
  a.open = open;
  a.account = account;
  a.table = const_cast<int32_t*>(table);
  hipLaunchKernelGGL(tables_free_kernel, dim3(static_cast<uint32_t>(n)), dim3(kRowThreads), 0, static_cast<hipStream_t>(stream), a, which);
  KVQ_LAUNCH_CHECK("kvq_tables_free");
  return KVQ_OK;
}
