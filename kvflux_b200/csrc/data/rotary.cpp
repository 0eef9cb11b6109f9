// RotaryTable and write_paged_kv_rotated (include/kvflux/v2/rotary.h).
#include "kvflux/v2/rotary.h"

#include <utility>

#include "runtime.h"

namespace kvflux::v2 {

RotaryTable::RotaryTable(std::size_t max_positions, std::size_t rotary_dim, double base, double position_scale,
                         bool interleaved, int device)
    : max_positions_(max_positions), rotary_dim_(rotary_dim), interleaved_(interleaved), device_(device) {
    if (max_positions == 0 || rotary_dim == 0 || rotary_dim % 2 != 0 || rotary_dim > UINT32_MAX) {
        throw std::invalid_argument("rotary table needs positions and a positive, even rotary_dim");
    }
    const std::size_t bytes =
        detail::mul_checked(detail::mul_checked(max_positions, rotary_dim, "rotary table"), sizeof(float), "rotary table");
    if (device < 0) throw std::invalid_argument("device ordinal must be non-negative");
    int count = 0;
    detail::cuda_check(cudaGetDeviceCount(&count), "cudaGetDeviceCount");
    if (device >= count) throw std::invalid_argument("GPU device index out of range");
    detail::DeviceGuard guard(device);
    void* table = nullptr;
    detail::cuda_check(cudaMalloc(&table, bytes), "allocate rotary table");
    table_ = static_cast<float*>(table);
    try {
        detail::check_kvfx(kvfx_rotary_table(table_, max_positions, static_cast<uint32_t>(rotary_dim), base,
                                             position_scale, device, nullptr),
                           "rotary table");
        detail::cuda_check(cudaStreamSynchronize(nullptr), "rotary table synchronize");
    } catch (...) {
        (void)cudaFree(table_);
        throw;
    }
}

RotaryTable::~RotaryTable() noexcept {
    int previous = 0;
    if (table_ != nullptr && cudaGetDevice(&previous) == cudaSuccess && cudaSetDevice(device_) == cudaSuccess) {
        (void)cudaFree(table_);
        (void)cudaSetDevice(previous);
    }
}

void write_paged_kv_rotated(PagedKVStorage& storage, const RotaryTable& table, const HeadNorms& norms,
                            const ProjectedTokens& tokens, std::size_t query_heads,
                            const std::vector<std::size_t>& positions, const SlotMapping& slot_mapping,
                            float* query_out_device) {
    if (slot_mapping.empty()) return;
    if (tokens.key == nullptr || tokens.value == nullptr ||
        (query_heads != 0 && (tokens.query == nullptr || query_out_device == nullptr))) {
        throw std::invalid_argument("Q, K, V and Q output device pointers are required");
    }
    const PagedKVLayout& layout = storage.layout();
    if (table.device() != storage.device()) {
        throw std::invalid_argument("rotary table and KV storage must be on one GPU");
    }
    if (table.rotary_dim() > layout.head_size()) throw std::invalid_argument("rotary_dim above the head size");
    if (positions.size() != slot_mapping.size()) throw std::invalid_argument("one position per slot is required");
    if (query_heads > UINT32_MAX) throw std::invalid_argument("too many query heads");
    detail::StorageRuntime& rt = storage.runtime();
    detail::check_slots(rt, layout, slot_mapping);
    for (const std::size_t p : positions) {
        if (p >= table.max_positions()) throw std::out_of_range("position beyond the rotary table");
    }
    const char* op = "rotated KV write";
    const std::size_t n = slot_mapping.size(), elem = layout.element_bytes();
    auto span = [&](std::size_t stride, std::size_t heads) {  // bytes from the first token's row to the last's end
        const std::size_t row = detail::mul_checked(heads, layout.head_size(), op);
        if (stride < row) throw std::invalid_argument("a stride is smaller than one token's heads");
        return detail::mul_checked(detail::mul_checked(n, stride, op) - (stride - row), elem, op);
    };
    const std::size_t k_bytes = span(tokens.key_stride, layout.num_kv_heads());
    const std::size_t v_bytes = span(tokens.value_stride, layout.num_kv_heads());
    const std::size_t q_bytes = query_heads != 0 ? span(tokens.query_stride, query_heads) : 0;
    const std::size_t out_bytes = detail::mul_checked(
        detail::mul_checked(detail::mul_checked(n, query_heads, op), layout.head_size(), op), sizeof(float), op);

    detail::DeviceGuard guard(storage.device());
    detail::require_device_pointer(tokens.key, storage.device(), "K");
    detail::require_device_pointer(tokens.value, storage.device(), "V");
    if (norms.query_weight != nullptr) {
        detail::require_device_pointer(norms.query_weight, storage.device(), "query norm weight");
    }
    if (norms.key_weight != nullptr) {
        detail::require_device_pointer(norms.key_weight, storage.device(), "key norm weight");
    }
    if (query_heads != 0) {
        detail::require_device_pointer(tokens.query, storage.device(), "Q");
        detail::require_device_pointer(query_out_device, storage.device(), "Q output");
    }
    // Nothing that is read may lie where the call writes.
    const std::size_t weight_bytes = layout.head_size() * sizeof(float);
    const std::pair<const void*, std::size_t> inputs[] = {
        {tokens.key, k_bytes},
        {tokens.value, v_bytes},
        {tokens.query, q_bytes},
        {norms.query_weight, norms.query_weight != nullptr ? weight_bytes : 0},
        {norms.key_weight, norms.key_weight != nullptr ? weight_bytes : 0},
        {table.device_table(), table.max_positions() * table.rotary_dim() * sizeof(float)},
    };
    for (const auto& [input, input_bytes] : inputs) {
        if (input_bytes == 0) continue;
        if (detail::overlaps(input, input_bytes, storage.key_base(), layout.total_bytes())) {
            throw std::invalid_argument("rotated KV write inputs must not lie in the KV cache");
        }
        if (out_bytes != 0 && detail::overlaps(query_out_device, out_bytes, input, input_bytes)) {
            throw std::invalid_argument("Q output must not overlap the inputs or the KV cache");
        }
    }
    if (out_bytes != 0 && detail::overlaps(query_out_device, out_bytes, storage.key_base(), layout.total_bytes())) {
        throw std::invalid_argument("Q output must not overlap the inputs or the KV cache");
    }
    const std::size_t bytes[2] = {n * sizeof(PhysicalSlot), n * sizeof(std::size_t)};
    const void* host[2] = {slot_mapping.data(), positions.data()};
    void* dev[2] = {nullptr, nullptr};
    rt.upload(host, bytes, 2, dev);
    const kvfx_rotary rotary{table.device_table(), table.max_positions(), static_cast<uint32_t>(table.rotary_dim()),
                             table.interleaved() ? 1u : 0u, norms.query_weight, norms.key_weight, norms.epsilon, 0};
    detail::check_kvfx(kvfx_write_rotated(&rt.cache, &rotary, tokens.query, tokens.key, tokens.value,
                                          tokens.query_stride, tokens.key_stride, tokens.value_stride,
                                          static_cast<uint32_t>(query_heads), static_cast<const uint64_t*>(dev[1]),
                                          static_cast<const uint64_t*>(dev[0]), n, query_out_device, nullptr),
                       op);
    rt.finish("rotated KV write synchronize");
}

}  // namespace kvflux::v2
