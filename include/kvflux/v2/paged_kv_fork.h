#pragma once
// Forks and compaction of sequences whose model keeps one PagedKVStorage per
// layer over one PhysicalBlockPool (see paged_kv_layers.h for what the layers
// must have in common): the page bookkeeping and one launch for all layers'
// copies. Synchronous on the legacy default stream. No counterpart in the
// reference, which copies one page of one layer at a time
// (include/kvflux/v2/paged_kv_storage.h:39) and never drops tokens.
#include "kvflux/v2/paged_kv_storage.h"
#include "kvflux/v2/sequence_state.h"

#include <cstddef>
#include <vector>

namespace kvflux::v2 {

// One child per request id, each with the source's tokens: full pages are
// shared (as SequenceState::fork_shared), a partial last page is copied to a
// page of the child's own, so that source and children append without
// copy-on-write. If the pool runs out of pages (CapacityError) or the copy
// fails, nothing has changed.
std::vector<SequenceState> fork_sequence(const std::vector<PagedKVStorage*>& layers, const SequenceState& source,
                                         const std::vector<RequestID>& children);

// Keeps only the tokens at the positions `keep` (strictly ascending, each
// below num_tokens()), in order, as positions 0 .. keep.size() - 1: leading
// pages that stay whole are kept as they are (shared ones included), the other
// kept tokens move to fresh pages, and the old pages lose this sequence's
// reference. K and V are moved as they are: keys that carry positions keep
// those of their writing. If the pool runs out of pages or the copy fails,
// nothing has changed. Throws invalid_argument where `keep` does not ascend,
// out_of_range for a position beyond the sequence. A BatchDecodeSession over
// the sequence must be refreshed.
void compact_sequence(const std::vector<PagedKVStorage*>& layers, SequenceState& sequence,
                      const std::vector<std::size_t>& keep);

} // namespace kvflux::v2
