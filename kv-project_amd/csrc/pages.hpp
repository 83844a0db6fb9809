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
// A step's description (int32 words on the device): a header of 8 words {sequences, items, split items,
// units per split, whether every sequence has one item, the most new
// tokens of one}, then 8 words per sequence {slot, tokens before, new tokens, first packed row, first
// item, first split item, open buffer before | after << 1} and one entry behind the last with the
// totals, then the page of every item.  An item is a block that the step's tokens touch.
#pragma once
#include "common.hpp"

namespace kvq {

constexpr int kStepHead = 8, kStepSeq = 8;
constexpr int kUnit = 64;                     // tokens of one decode unit

enum { kCodeInt8 = 0, kCodeE4M3 = 1 };

struct StepSeq {
  int slot, pos0, count, row0, item0, split0, bufs;
};

__device__ __forceinline__ StepSeq step_seq(const int* step, int b) {
  const int* e = step + kStepHead + kStepSeq * b;
  return {e[0], e[1], e[2], e[3], e[4], e[5], e[6]};
}

// The last of n sequences whose word (at first[i * stride]) is not above `value`: 64 at a time, one memory round trip
// each instead of one per halving.  By whole wavefronts, `value` the same in all lanes.
__device__ __forceinline__ int last_not_above(const int* first, int stride, int n, int value) {
  const int lane = threadIdx.x & 63;
  int count = 0;
  for (int i = 0; i < n; i += 64) {
    const int x = i + lane < n ? first[(i + lane) * stride] : 0x7fffffff;
    const int c = __popcll(__builtin_amdgcn_ballot_w64(x <= value));
    count += c;
    if (c < 64) break;
  }
  return count - 1;
}

// The sequence whose range [first, next first) of word `w` holds i (ranges may be empty).
__device__ __forceinline__ int step_find(const int* step, int n, int w, int i) {
  return __builtin_amdgcn_readfirstlane(last_not_above(step + kStepHead + w, kStepSeq, n, i));
}

}  // namespace kvq
