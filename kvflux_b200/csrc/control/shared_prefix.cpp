// plan_shared_prefixes (include/kvflux/v2/shared_prefix.h).
#include "kvflux/v2/shared_prefix.h"

#include <algorithm>
#include <stdexcept>

namespace kvflux::v2 {

namespace {

// Shorter shared prefixes are cheaper to read again than to share.
constexpr std::size_t kMinSharedPages = 8;

}  // namespace

std::vector<PrefixGroup> plan_shared_prefixes(const std::vector<const SequenceState*>& sequences) {
    std::vector<PrefixGroup> groups;
    if (sequences.empty()) return groups;
    for (const SequenceState* s : sequences) {
        if (s == nullptr) throw std::invalid_argument("null sequence in batch");
        if (!s->block_table().shares_pool_with(sequences.front()->block_table())) {
            throw std::invalid_argument("batch sequences must share one physical pool");
        }
    }
    const std::size_t block = sequences.front()->block_size();
    auto whole_pages = [](const SequenceState& s) { return s.num_tokens() / s.block_size(); };
    auto close = [&](std::size_t rows, std::size_t pages) {
        if (pages < kMinSharedPages || rows < 2) pages = 0;
        if (pages == 0 && !groups.empty() && groups.back().prefix_tokens == 0) {
            groups.back().rows += rows;
        } else {
            groups.push_back({rows, pages * block});
        }
    };
    std::size_t rows = 1, shared = whole_pages(*sequences.front());
    for (std::size_t r = 1; r < sequences.size(); ++r) {
        const SequenceState &last = *sequences[r - 1], &next = *sequences[r];
        const std::size_t common =
            last.block_table().common_entries(next.block_table(), std::min(shared, whole_pages(next)));
        // Saved page reads with this sequence, and without it.
        if (common >= kMinSharedPages && rows * common >= (rows - 1) * shared) {
            ++rows;
            shared = common;
        } else {
            close(rows, shared);
            rows = 1;
            shared = whole_pages(next);
        }
    }
    close(rows, shared);
    return groups;
}

}  // namespace kvflux::v2
