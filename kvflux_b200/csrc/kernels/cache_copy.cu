// Copies inside the paged caches of a layer batch: whole pages (forks of
// requests) and single tokens' rows (compaction after an eviction).
//
//   pages  K_l[dst_i][:][:][:] = K_l[src_i][:][:][:], V alike
//   slots  K_l[dst_i / bs][h][dst_i % bs][:] = K_l[src_i / bs][h][src_i % bs][:]
//
// for every layer l. Both are bit copies bounded by HBM (each byte read once
// and written once), so they move 16-byte vectors where the shapes allow and
// never look at the element type. One launch covers every layer: blockIdx.y
// is the layer, whose bases come from the kernel parameters, and blockIdx.z
// the cache (K or V), which doubles the CTAs of a small copy. Work is a flat
// range of vectors, so that pages of any size fill their CTAs, two vectors a
// thread: small CTAs end evenly. B200, in a graph: 8190 tokens in 16 layers
// 164 us, 6.56 TB/s read and written (1.00 of the plain copy rate; 165 / 173 us
// with 4 / 8 vectors), 96 pages from 24 in 32 layers 42.8 us (201 MB written,
// the repeated sources read from the L2; 42.4 / 43.3), 8 pages in one layer
// 1.8 us (2.2 / 2.9).
#include <algorithm>

#include "common.cuh"
#include "launch.h"

namespace kvfx {
namespace {

constexpr int kThreads = 256;
constexpr int kPer = 2;  // vectors in flight per thread before its first store

template <int VB>
__global__ void __launch_bounds__(kThreads) copy_pages_kernel(const __grid_constant__ LayerBases bases,
                                                              const uint64_t* __restrict__ src,
                                                              const uint64_t* __restrict__ dst, uint32_t total,
                                                              uint32_t page_vecs, FastDiv div_page,
                                                              uint64_t num_blocks, unsigned* status) {
    using V = typename Vec<VB>::T;
    pdl_allow_next();
    pdl_wait();  // launched as a dependent: the previous kernel's writes first
    V* base = reinterpret_cast<V*>(blockIdx.z == 0 ? bases.k[blockIdx.y] : bases.v[blockIdx.y]);
    const uint32_t e0 = blockIdx.x * (kThreads * kPer) + threadIdx.x;
    V x[kPer];
    uint64_t to[kPer];
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
        const uint32_t e = e0 + j * kThreads;
        to[j] = ~0ull;
        if (e >= total) continue;
        const uint32_t i = fast_div(e, div_page);
        const uint32_t c = e - i * page_vecs;
        const uint64_t s = __ldg(src + i), d = __ldg(dst + i);
        if (s >= num_blocks || d >= num_blocks) {
            raise_flag(status, KVFX_FLAG_BAD_INDEX);
            continue;
        }
        x[j] = base[s * page_vecs + c];
        to[j] = d * page_vecs + c;
    }
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
        if (to[j] != ~0ull) base[to[j]] = x[j];
    }
}

// Vector e of a slot copy: tokens in groups of 16, e = ((group * heads + h) *
// 16 + token in group) * vpr + c. Consecutive destination slots of a page are
// consecutive rows of one head, so a group that fills a 16-token page stores
// one contiguous run per head, and kept neighbours load as runs too.
constexpr uint32_t kSlotGroup = 16;

template <int VB>
__global__ void __launch_bounds__(kThreads) copy_slots_kernel(
    const __grid_constant__ LayerBases bases, const uint64_t* __restrict__ src, const uint64_t* __restrict__ dst,
    uint32_t n, uint32_t total, uint32_t heads, uint32_t vpr, uint32_t bs, FastDiv div_vpr, FastDiv div_heads,
    uint64_t slot_count, unsigned* status) {
    using V = typename Vec<VB>::T;
    pdl_allow_next();
    pdl_wait();  // launched as a dependent: the previous kernel's writes first
    V* base = reinterpret_cast<V*>(blockIdx.z == 0 ? bases.k[blockIdx.y] : bases.v[blockIdx.y]);
    const uint32_t e0 = blockIdx.x * (kThreads * kPer) + threadIdx.x;
    const bool pow2 = (bs & (bs - 1)) == 0;  // every usual page: no 64-bit division
    const int shift = 31 - __clz(static_cast<int>(bs));
    V x[kPer];
    uint64_t to[kPer];
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
        const uint32_t e = e0 + j * kThreads;
        to[j] = ~0ull;
        if (e >= total) continue;
        const uint32_t row = fast_div(e, div_vpr);
        const uint32_t c = e - row * vpr;
        const uint32_t gh = row / kSlotGroup;
        const uint32_t group = fast_div(gh, div_heads);
        const uint32_t h = gh - group * heads;
        const uint32_t i = group * kSlotGroup + row % kSlotGroup;
        if (i >= n) continue;
        const uint64_t s = __ldg(src + i), d = __ldg(dst + i);
        if (s >= slot_count || d >= slot_count) {
            raise_flag(status, KVFX_FLAG_BAD_INDEX);
            continue;
        }
        const uint64_t sp = pow2 ? s >> shift : s / bs, dp = pow2 ? d >> shift : d / bs;
        x[j] = base[((sp * heads + h) * bs + (s - sp * bs)) * vpr + c];
        to[j] = ((dp * heads + h) * bs + (d - dp * bs)) * vpr + c;
    }
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
        if (to[j] != ~0ull) base[to[j]] = x[j];
    }
}

// Widest vector that divides `bytes` and every layer's bases.
uint32_t layers_vector_width(const CacheView* layers, uint32_t num_layers, uint64_t bytes) {
    uint32_t width = 16;
    for (uint32_t l = 0; l < num_layers; ++l) {
        const void* ptrs[2] = {layers[l].k, layers[l].v};
        width = std::min(width, vector_width(bytes, ptrs, 2));
    }
    return width;
}

// Vectors one launch covers at most (32-bit indices, with room for padding).
constexpr uint64_t kMaxVecs = 1ull << 30;

template <int VB>
cudaError_t pages_vb(const CacheView& c, const LayerBases& bases, uint32_t num_layers, const uint64_t* src,
                     const uint64_t* dst, uint64_t n, unsigned* status, cudaStream_t s) {
    const uint64_t page_vecs = c.page_bytes / VB;
    if (page_vecs > kMaxVecs) return cudaErrorInvalidValue;  // a page of 1 GiB and more
    const uint64_t step = std::max<uint64_t>(1, kMaxVecs / page_vecs);
    for (uint64_t i = 0; i < n; i += step) {
        const uint64_t total = std::min(step, n - i) * page_vecs;
        const dim3 grid(static_cast<uint32_t>(ceil_div(total, kThreads * kPer)), num_layers, 2);
        const cudaError_t e = launch_dependent(
            copy_pages_kernel<VB>, grid, dim3(kThreads), s, bases, src + i, dst + i, static_cast<uint32_t>(total),
            static_cast<uint32_t>(page_vecs), make_fastdiv(static_cast<uint32_t>(page_vecs)), c.num_blocks, status);
        if (e != cudaSuccess) return e;
    }
    return cudaSuccess;
}

template <int VB>
cudaError_t slots_vb(const CacheView& c, const LayerBases& bases, uint32_t num_layers, const uint64_t* src,
                     const uint64_t* dst, uint64_t n, unsigned* status, cudaStream_t s) {
    const uint64_t vpr = c.row_bytes / VB;
    const uint64_t group_vecs = vpr * c.heads * kSlotGroup;
    if (group_vecs > kMaxVecs) return cudaErrorInvalidValue;  // 16 tokens of 1 GiB and more
    const uint64_t step = std::max<uint64_t>(1, kMaxVecs / group_vecs) * kSlotGroup;
    for (uint64_t i = 0; i < n; i += step) {
        const uint64_t count = std::min(step, n - i);
        const uint64_t total = ceil_div(count, kSlotGroup) * group_vecs;
        const dim3 grid(static_cast<uint32_t>(ceil_div(total, kThreads * kPer)), num_layers, 2);
        const cudaError_t e = launch_dependent(
            copy_slots_kernel<VB>, grid, dim3(kThreads), s, bases, src + i, dst + i, static_cast<uint32_t>(count),
            static_cast<uint32_t>(total), c.heads, static_cast<uint32_t>(vpr), c.bs,
            make_fastdiv(static_cast<uint32_t>(vpr)), make_fastdiv(c.heads), c.slot_count, status);
        if (e != cudaSuccess) return e;
    }
    return cudaSuccess;
}

LayerBases bases_of(const CacheView* layers, uint32_t num_layers) {
    LayerBases bases{};
    for (uint32_t l = 0; l < num_layers; ++l) {
        bases.k[l] = layers[l].k;
        bases.v[l] = layers[l].v;
    }
    return bases;
}

}  // namespace

cudaError_t launch_copy_pages(const CacheView* layers, uint32_t num_layers, const uint64_t* src, const uint64_t* dst,
                              uint64_t n, unsigned* status, cudaStream_t s) {
    const CacheView& c = layers[0];
    const LayerBases bases = bases_of(layers, num_layers);
    switch (layers_vector_width(layers, num_layers, c.page_bytes)) {
    case 16: return pages_vb<16>(c, bases, num_layers, src, dst, n, status, s);
    case 8: return pages_vb<8>(c, bases, num_layers, src, dst, n, status, s);
    case 4: return pages_vb<4>(c, bases, num_layers, src, dst, n, status, s);
    case 2: return pages_vb<2>(c, bases, num_layers, src, dst, n, status, s);
    default: return pages_vb<1>(c, bases, num_layers, src, dst, n, status, s);
    }
}

cudaError_t launch_copy_slots(const CacheView* layers, uint32_t num_layers, const uint64_t* src, const uint64_t* dst,
                              uint64_t n, unsigned* status, cudaStream_t s) {
    const CacheView& c = layers[0];
    const LayerBases bases = bases_of(layers, num_layers);
    switch (layers_vector_width(layers, num_layers, c.row_bytes)) {
    case 16: return slots_vb<16>(c, bases, num_layers, src, dst, n, status, s);
    case 8: return slots_vb<8>(c, bases, num_layers, src, dst, n, status, s);
    case 4: return slots_vb<4>(c, bases, num_layers, src, dst, n, status, s);
    case 2: return slots_vb<2>(c, bases, num_layers, src, dst, n, status, s);
    default: return slots_vb<1>(c, bases, num_layers, src, dst, n, status, s);
    }
}

}  // namespace kvfx
