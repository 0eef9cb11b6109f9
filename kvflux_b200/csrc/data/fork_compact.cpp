// fork_sequence and compact_sequence (include/kvflux/v2/paged_kv_fork.h): page
// bookkeeping on new SequenceStates, which replace or join the old ones only
// once every layer's copy (one kvfx_copy_pages / kvfx_copy_slots launch) is done.
#include <algorithm>
#include <utility>

#include "kvflux/v2/paged_kv_fork.h"
#include "runtime.h"

namespace kvflux::v2 {

namespace {

// The layers of a call: non-null, alike, and on the sequence's pool.
const PagedKVStorage& check(const std::vector<PagedKVStorage*>& layers, const SequenceState& sequence,
                            const char* op) {
    const std::vector<const PagedKVStorage*> view(layers.begin(), layers.end());
    const PagedKVStorage& first = detail::check_layers(view.data(), view.size(), op);
    for (const PagedKVStorage* l : layers) {
        if (!l->uses_pool(sequence.block_table()) || sequence.block_size() != l->layout().block_size()) {
            throw std::invalid_argument("sequence and KV storage must use one physical pool");
        }
    }
    return first;
}

using CopyFn = int (*)(const kvfx_cache*, uint32_t, const uint64_t*, const uint64_t*, uint64_t, void*);

// Uploads the ids, copies in every layer and waits.
void copy_in_layers(const std::vector<PagedKVStorage*>& layers, const std::vector<uint64_t>& src,
                    const std::vector<uint64_t>& dst, CopyFn copy, const char* op) {
    const PagedKVStorage& first = *layers.front();
    detail::DeviceGuard guard(first.device());
    detail::StorageRuntime& rt = first.runtime();
    try {
        const std::size_t bytes[2] = {src.size() * sizeof(uint64_t), dst.size() * sizeof(uint64_t)};
        const void* host[2] = {src.data(), dst.data()};
        void* dev[2] = {nullptr, nullptr};
        rt.upload(host, bytes, 2, dev);
        const std::vector<const PagedKVStorage*> view(layers.begin(), layers.end());
        const std::vector<kvfx_cache> caches = detail::layer_descriptors(view.data(), view.size());
        detail::check_kvfx(copy(caches.data(), static_cast<uint32_t>(caches.size()), static_cast<const uint64_t*>(dev[0]),
                                static_cast<const uint64_t*>(dev[1]), src.size(), nullptr),
                           op);
        rt.finish(op);
    } catch (...) {
        // Work already queued must finish before the caller's pages are reused.
        (void)cudaStreamSynchronize(nullptr);
        throw;
    }
}

}  // namespace

std::vector<SequenceState> fork_sequence(const std::vector<PagedKVStorage*>& layers, const SequenceState& source,
                                         const std::vector<RequestID>& children) {
    (void)check(layers, source, "fork");
    const std::size_t bs = source.block_size(), full = source.num_tokens() / bs, rest = source.num_tokens() % bs;
    std::vector<SequenceState> out;
    out.reserve(children.size());
    std::vector<uint64_t> src, dst;
    for (const RequestID id : children) {
        out.push_back(source.fork_prefix(id, full));  // pages go back if anything below throws
        if (rest == 0) continue;
        out.back().append_tokens(rest);
        src.push_back(source.physical_block_id(full));
        dst.push_back(out.back().physical_block_id(full));
    }
    for (const std::vector<uint64_t>* ids : {&src, &dst}) {
        for (const uint64_t id : *ids) {
            if (id >= layers.front()->layout().num_blocks()) throw std::out_of_range("fork block out of range");
        }
    }
    if (!src.empty()) copy_in_layers(layers, src, dst, kvfx_copy_pages, "fork");
    return out;
}

void compact_sequence(const std::vector<PagedKVStorage*>& layers, SequenceState& sequence,
                      const std::vector<std::size_t>& keep) {
    const PagedKVStorage& first = check(layers, sequence, "compaction");
    for (std::size_t i = 0; i < keep.size(); ++i) {
        if (i != 0 && keep[i] <= keep[i - 1]) throw std::invalid_argument("kept positions must ascend");
        if (keep[i] >= sequence.num_tokens()) throw std::out_of_range("kept position beyond the sequence");
    }
    if (keep.size() == sequence.num_tokens()) return;
    const std::size_t bs = sequence.block_size();
    std::size_t same = 0;  // leading tokens that stay where they are
    while (same < keep.size() && keep[same] == same) ++same;
    const std::size_t pages = same / bs;
    SequenceState next = sequence.fork_prefix(sequence.request_id(), pages);
    next.append_tokens(keep.size() - pages * bs);
    std::vector<PhysicalBlockID> from(sequence.num_allocated_blocks()), to(next.num_allocated_blocks());
    if (!from.empty()) sequence.copy_physical_block_ids(from.data());
    if (!to.empty()) next.copy_physical_block_ids(to.data());
    for (const std::vector<PhysicalBlockID>* ids : {&from, &to}) {
        for (const PhysicalBlockID id : *ids) {
            if (id >= first.layout().num_blocks()) throw std::out_of_range("compaction block out of range");
        }
    }
    std::vector<uint64_t> src, dst;
    src.reserve(keep.size() - pages * bs);
    dst.reserve(keep.size() - pages * bs);
    for (std::size_t i = pages * bs; i < keep.size(); ++i) {
        src.push_back(from[keep[i] / bs] * bs + keep[i] % bs);
        dst.push_back(to[i / bs] * bs + i % bs);
    }
    if (!src.empty()) copy_in_layers(layers, src, dst, kvfx_copy_slots, "compaction");
    sequence = std::move(next);
}

}  // namespace kvflux::v2
