#pragma once
// Batch decode attention over sequences that share leading pages (prefix-cache
// hits, forks of one prompt). No counterpart in the reference, whose
// paged_attention_batch (include/kvflux/v2/paged_attention.h:30) re-reads the
// shared pages for every sequence.
#include "kvflux/v2/paged_kv_storage.h"
#include "kvflux/v2/sequence_state.h"

#include <cstddef>
#include <vector>

namespace kvflux::v2 {

// A run of consecutive sequences of a batch whose first prefix_tokens
// positions (whole pages) lie in the same physical pages.
struct PrefixGroup {
    std::size_t rows;
    std::size_t prefix_tokens;
};

// Cuts a batch into such runs, in order: a run grows by its next sequence as
// long as the pages it saves reading ((rows - 1) x shared pages) do not
// shrink; runs that would share fewer than 8 pages share none, and consecutive
// ones of those are one group. Sequences that should share belong next to each
// other, without one between them that shares less: a lone sequence saves
// nothing, so it takes any neighbour that it shares 8 pages with. All sequences
// must be non-null and of one pool (invalid_argument).
std::vector<PrefixGroup> plan_shared_prefixes(const std::vector<const SequenceState*>& sequences);

// paged_attention_batch (same arguments, checks, exceptions, synchronous
// legacy-default-stream contract, and results within the same tolerances) that
// reads the pages each run of plan_shared_prefixes shares once for the run.
void paged_attention_batch_shared(const PagedKVStorage& storage,
                                  const std::vector<const SequenceState*>& sequences,
                                  const float* query_device, float* output_device,
                                  std::size_t query_heads);

} // namespace kvflux::v2
