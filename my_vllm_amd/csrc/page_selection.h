// Sizes that the page selection and the attention over selected pages share.
//
// Workspace: [arrival counters of the selection][of the attention][partials of
// the attention][score keys of the selection].  The counters lie at one place
// whatever the sizes: they are zero between launches, of any sizes.  The partials
// come before the keys: the attention knows its own sizes only.
#pragma once

#include <cstdint>

namespace mva {

constexpr int kPageTokens = 16;
constexpr int kMaxQueryGroup = 16;

// (row, KV head) pairs of a launch whose workgroups count themselves in.
constexpr int kSelectionCounters = 1024;
constexpr int64_t kSelectionHeaderBytes = 2 * kSelectionCounters * 4;

inline int64_t align_up256(int64_t x) { return (x + 255) & ~int64_t(255); }

// Whether a selection of `num_selected` pages a row can be made at all.
inline bool selection_sizes_ok(int64_t num_seqs, int hq, int hkv, int64_t num_selected) {
  return num_seqs >= 0 && num_seqs <= 0x7fffffffLL && hkv > 0 && hq > 0 && hq % hkv == 0 && hq / hkv <= kMaxQueryGroup &&
         num_seqs * hq <= 0x7fffffffLL && num_selected > 0 && num_selected <= (1 << 24);
}

// Bytes kept for the attention's partials; they do not fall as any of the sizes grows.
int64_t selection_part_bytes(int64_t num_seqs, int hq, int64_t num_selected);

}  // namespace mva
