#pragma once
// Per-head RMS norms and rotary positions of new tokens' Q and K, in the same
// pass as their paged KV write. No counterpart in the reference, whose
// write_paged_kv (include/kvflux/v2/paged_kv_write.h:14-15) takes K and V as
// they go into the cache.
#include "kvflux/v2/paged_kv_storage.h"

#include <cstddef>
#include <vector>

namespace kvflux::v2 {

// Cosines and sines of max_positions positions on one GPU: angle i of position
// p is p * position_scale * base^(-2i / rotary_dim), computed in FP64. The
// first rotary_dim dimensions of a head are turned in pairs (i, i + rotary_dim
// / 2), or (2i, 2i + 1) when interleaved.
class RotaryTable {
public:
    RotaryTable(std::size_t max_positions, std::size_t rotary_dim, double base = 10000.0,
                double position_scale = 1.0, bool interleaved = false, int device = 0);
    ~RotaryTable() noexcept;
    RotaryTable(const RotaryTable&) = delete;
    RotaryTable& operator=(const RotaryTable&) = delete;

    std::size_t max_positions() const noexcept { return max_positions_; }
    std::size_t rotary_dim() const noexcept { return rotary_dim_; }
    bool interleaved() const noexcept { return interleaved_; }
    int device() const noexcept { return device_; }
    // Device float[max_positions][rotary_dim]: a row's cosines, then its sines.
    const float* device_table() const noexcept { return table_; }

private:
    std::size_t max_positions_, rotary_dim_;
    bool interleaved_;
    int device_;
    float* table_ = nullptr;
};

// Norm weights (device float[head_size], null for no norm) and the epsilon
// added to the mean square.
struct HeadNorms {
    const float* query_weight = nullptr;
    const float* key_weight = nullptr;
    float epsilon = 1e-6f;
};

// New tokens' projections on the device, in the storage's dtype: token t's
// heads are contiguous from query + t * query_stride on (elements; likewise
// key and value), so the three may be slices of one buffer.
struct ProjectedTokens {
    const void* query;
    const void* key;
    const void* value;
    std::size_t query_stride, key_stride, value_stride;
};

// Norms and rotates Q and K, writes K and V to `slot_mapping` as
// write_paged_kv does (same slot checks), and Q in FP32 to query_out_device
// [tokens][query_heads][head_size], ready for the attention calls. positions:
// one per token. query_heads may be 0 (Q is then not looked at). Synchronous
// on the legacy default stream; an empty mapping returns at once. Throws
// invalid_argument for null or foreign-device pointers, a table of another
// device or wider than the head, strides below a token's heads, a position
// count other than the slots', an input (norm weights among them) in the
// cache, and query_out_device overlapping an input or the cache; out_of_range
// for a slot or position out of range.
void write_paged_kv_rotated(PagedKVStorage& storage, const RotaryTable& table, const HeadNorms& norms,
                            const ProjectedTokens& tokens, std::size_t query_heads,
                            const std::vector<std::size_t>& positions, const SlotMapping& slot_mapping,
                            float* query_out_device);

} // namespace kvflux::v2
