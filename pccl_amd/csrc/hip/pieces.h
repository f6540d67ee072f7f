// pieces.h -- how a call that is too large for one launch is cut into several (host only; nothing of HIP in here).
#pragma once

#include <algorithm>

namespace pccl_host {

// Calls f(first, n) for [0, total) in pieces of `most`, the last one shorter, until one of them returns something other than 0;
// returns that.  All in 64 bits: a 32-bit start would pass its largest value behind the last piece of a total near 2^31.
template <class F>
int in_pieces(long total, long most, F &&f) {
  for (long first = 0; first < total; first += most) {
    const int rc = f(first, std::min(most, total - first));
    if (rc != 0) return rc;
  }
  return 0;
}

// Tokens of a sequence, `most` of them at most, that `entries` pages of `page_tokens` have room for; entries may be anything from 0.
inline long tokens_in_pages(long most, long entries, long page_tokens) {
  return entries > most / page_tokens ? most : entries * page_tokens;
}

}  // namespace pccl_host
