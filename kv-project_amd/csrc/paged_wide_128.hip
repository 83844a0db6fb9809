// paged_wide.hpp's kernels at head_dim 128: a source of its own, so that both compile side by side
#include "paged_wide.hpp"

void kvq::launch_wide_128(const WideArgs& a, int page, int code, bool bf16, int waves, int64_t items, int64_t merges, int64_t most_parts,
                          hipStream_t stream) {
  launch_wide<128>(a, page, code, bf16, waves, items, merges, most_parts, stream);
}
