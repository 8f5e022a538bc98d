// What the optimizers' steps share.
#pragma once

#include <algorithm>
#include <utility>
#include <vector>

#include "common.h"

namespace strata {

// Ranges of memory (first byte, one past the last) that a call writes and reads: the written ones may overlap nothing.
inline int check_ranges(const std::string& name, std::vector<std::pair<uintptr_t, uintptr_t>>& written,
                        const std::vector<std::pair<uintptr_t, uintptr_t>>& read) {
  std::sort(written.begin(), written.end());
  for (size_t i = 1; i < written.size(); ++i)
    if (written[i].first < written[i - 1].second)
      return fail(STRATA_HIP_EINVAL, name + ": two of the tensors to update overlap");
  for (const auto& r : read) {  // the ranges written are disjoint: the last one that starts before r ends
    auto w = std::lower_bound(written.begin(), written.end(), std::make_pair(r.second, (uintptr_t)0));
    if (w != written.begin() && (--w)->second > r.first)
      return fail(STRATA_HIP_EINVAL, name + ": a gradient overlaps a tensor to update");
  }
  return STRATA_HIP_OK;
}

}  // namespace strata
