// The paged 8-bit cache shared by its kernels: layouts, the step description and the codes.
//
// A sequence's tokens lie in blocks of P tokens (32, 64 or 128).  A full block is one page, shared by
// any number of sequences: per KV head P x D codes of 8 bits for the keys (token major) and D x P for
// the values (channel major, the order in which a probability row multiplies them), with one float32
// scale each.  The open block of a sequence stays in 16 bits in one of its slot's two open buffers,
// laid out like a page; a step that fills a block and opens the next one writes the other buffer, so
// what the full block was cut from stays, and a step can be run again.
//
//   kc (pages, H, P, D) bytes   vc (pages, H, D, P) bytes   sc (pages, H, 2) float: key, value scale
//   ko (slots, 2, H, P, D)      vo (slots, 2, H, D, P)      16-bit elements of the model's type
//   table (slots, max_blocks) int32: the page of each full block
//
// A step's description (int32 words on the device): a header of 12 words {sequences, items, split items,
// units per split, whether every sequence has one item, the most new tokens of one, the most of a run, the
// tokens of all split items, runs, first word of the items' pages, whether results are joined of several items,
// whether every run is one item}, then 8 words per sequence {slot, tokens
// before, new tokens, first packed row, first item, its run, open buffer before | after << 1, 1 + the run of its
// shared front or 0} and one entry behind the last with the totals, then the runs, then the page of every item.
// An item is a block that the step's tokens touch.
//
// A run is what a decode reads once for a range of packed rows, in split items of so many units: a sequence
// (or what is its own of it), or the pages that neighbouring sequences of the step share in front, for the rows of
// all of them.  12 words: {slot whose table row names the pages, first packed row, tokens, first unit, end,
// first split item, tokens of the split items before, sequence or -1, and of a sequence its tokens before, its
// open buffer, 1 + the run of its shared front or 0; split items}, and an entry behind the last.
#pragma once
#include "common.hpp"

namespace kvq {

constexpr int kStepHead = 12, kStepSeq = 8, kStepRun = 12;
constexpr int kUnit = 64;                     // tokens of one decode unit

enum { kCodeInt8 = 0, kCodeE4M3 = 1 };

struct StepSeq {
  int slot, pos0, count, row0, item0, run, bufs, front;
};
struct StepRun {
  int slot, row0, tokens, u0, u1, split0, base, seq, pos0, open, front, items;
};

__device__ __forceinline__ StepSeq step_seq(const int* step, int b) {
  const int* e = step + kStepHead + kStepSeq * b;
  return {e[0], e[1], e[2], e[3], e[4], e[5], e[6], e[7]};
}
__device__ __forceinline__ const int* step_runs(const int* step, int n) { return step + kStepHead + kStepSeq * (n + 1); }
__device__ __forceinline__ StepRun step_run(const int* runs, int i) {
  const int* e = runs + kStepRun * i;
  return {e[0], e[1], e[2], e[3], e[4], e[5], e[6], e[7], e[8], e[9], e[10], e[11]};
}

// The last of n sequences whose word (at first[i * stride]) is not above `value`: 256 at a time, one memory round trip
// each instead of one per halving.  By whole wavefronts, `value` the same in all lanes.
__device__ __forceinline__ int last_not_above(const int* first, int stride, int n, int value) {
  const int lane = threadIdx.x & 63;
  int count = 0;
  for (int i = 0; i < n; i += 256) {
    int x[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int at = i + 64 * k + lane;
      x[k] = first[(at < n ? at : n - 1) * stride];
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) count += __popcll(__builtin_amdgcn_ballot_w64(i + 64 * k + lane < n && x[k] <= value));
    if (count < i + 256) break;
  }
  return count - 1;
}

// The sequence whose range [first, next first) of word `w` holds i (ranges may be empty).
__device__ __forceinline__ int step_find(const int* step, int n, int w, int i) {
  return __builtin_amdgcn_readfirstlane(last_not_above(step + kStepHead + w, kStepSeq, n, i));
}

}  // namespace kvq
