// Batch decode over groups of rows that share a prefix (kvfx_decode_shared).
//
// A row's softmax over its positions is split at the end of its group's
// prefix, and each side further; a piece with running maximum m, sum l and
// unnormalised O joins the others by
//     M = max m,  L = sum l 2^(m - M),  o = (sum O 2^(m - M)) / L.
// One to three launches, each a programmatic dependent of the one before it:
//   prefix  (prefix.cu)   the groups' shared pages, once per 128 query rows;
//   tail    (decode.cu)   each row's own pages behind them;
//   merge   (below)       the pieces of every (row, query head).
// Where no row has more than one split of its own, the tail's CTAs join it
// with the prefix's pieces and write O ("fused"), and the merge is left out;
// where the rows are short and few, the tail reads all of their pages, shared
// ones too ("direct"), and is the only launch. make_plan has the rules.
// The workspace holds the pieces only, so nothing in it outlives a call.
#include <algorithm>
#include <cmath>

#include "common.cuh"
#include "launch.h"

namespace kvfx {
namespace {

constexpr int kMergeWarps = 4;
constexpr uint32_t kFirstCtas = 1024;  // about one wave
constexpr uint32_t kAhead = 8;  // pieces' O in flight

struct MergeParams {
    PrefixGroups groups;
    const uint64_t* lens;
    float* o;
    PrefixPieces pieces;   // prefix segments
    const float* tail;     // tail splits: [row][heads x chunks][split][8][hd + 2]
    uint64_t max_len, max_blocks;
    uint32_t q_heads, kv_heads, q_group, chunks;
    uint32_t pages_per_split, max_splits;
    unsigned* status;
};

// One warp per (row, query head); lane l holds dims 2l, 2l + 1 (and 64 more).
template <int HD>
__global__ void __launch_bounds__(kMergeWarps * 32) merge_kernel(const __grid_constant__ MergeParams p) {
    constexpr int kV = HD / 64;  // float2 per lane
    pdl_allow_next();
    const int lane = threadIdx.x & 31;
    const uint32_t id = blockIdx.x * kMergeWarps + (threadIdx.x >> 5);
    const uint32_t row = id / p.q_heads, j = id - row * p.q_heads;
    // Nothing before the wait below reads what the launches ahead write (the
    // lengths are older than both: see prefix.cu and the tail's order).
    const bool inside = row < p.groups.rows();
    const uint64_t len = inside ? __ldg(p.lens + row) : 0;
    if (len == 0) {  // padding
        pdl_wait();
        return;
    }
    const uint32_t g = p.groups.of_row(row);
    const uint32_t first = p.groups.pages[g];
    const uint64_t npages = ceil_div(len, 16);
    if (len > p.max_len || npages > p.max_blocks || len < static_cast<uint64_t>(first) * 16) {
        if (lane == 0) raise_flag(p.status, KVFX_FLAG_BAD_INDEX);
        pdl_wait();
        return;
    }
    // The row's pieces in order: its prefix segments, then its own splits.
    const uint32_t kh = j / p.q_group, gq = j - kh * p.q_group;
    uint32_t n_seg;
    uint64_t seg_row;  // first segment's row of part_o
    p.pieces.of_row(p.groups, g, row, kh, gq, p.q_group, &seg_row, &n_seg);
    const uint32_t own_pages = static_cast<uint32_t>(npages) - first;
    const uint32_t n = n_seg + (own_pages + p.pages_per_split - 1) / p.pages_per_split;
    const uint64_t unit = static_cast<uint64_t>(row) * (p.kv_heads * p.chunks) + kh * p.chunks + gq / 8;
    const float* tail = p.tail + (unit * p.max_splits * 8 + gq % 8) * (HD + 2);

    float M = -INFINITY, L = 0.f;
    float2 acc[kV];
#pragma unroll
    for (int v = 0; v < kV; ++v) acc[v] = make_float2(0.f, 0.f);
    float2* out = reinterpret_cast<float2*>(p.o + (static_cast<uint64_t>(row) * p.q_heads + j) * HD);
    // 32 pieces a pass, one a lane for (m, l) and the weights. A pass before
    // the wait reads this row's own output in place of a piece and forgets it:
    // it brings the loop's code and the kernel's parameters into the caches
    // while the launches ahead run (they stream more K and V than the L2
    // holds, so what is missing here would come from HBM, line after line).
    // (Only the first CTAs: the later ones find everything there.)
    uint32_t warm, base = 0;
    asm volatile("mov.u32 %0, 0;" : "=r"(warm) : "r"(n));  // unknown to the compiler: one copy of the loop; n is there
    if (blockIdx.x >= kFirstCtas) {
        warm = 1;
        pdl_wait();
    }
#pragma unroll 1
    do {
        const uint32_t here = warm != 0 ? min(32u, n - base) : 1u;
        const uint32_t i = base + lane;
        const uint64_t r = seg_row + static_cast<uint64_t>(i) * 128;
        const float* split = tail + static_cast<int64_t>(static_cast<int32_t>(i - n_seg)) * 8 * (HD + 2);
        const float* o = i < n_seg ? p.pieces.part_o + r * HD : split;
        const float* at = i < n_seg ? p.pieces.part_ml + r * 2 : split + HD;
        if (warm == 0) o = at = reinterpret_cast<const float*>(out);
        float2 ml = make_float2(-INFINITY, 0.f);
        if (lane < here) ml = __ldcg(reinterpret_cast<const float2*>(at));
        float m_new = ml.x;
#pragma unroll
        for (int s = 16; s > 0; s >>= 1) m_new = fmaxf(m_new, __shfl_xor_sync(0xffffffffu, m_new, s));
        m_new = fmaxf(m_new, M);
        const float keep = M == -INFINITY ? 0.f : exp2f(M - m_new);
        M = m_new;
        // A piece whose scores are all -inf weighs nothing, whatever its O holds.
        const float w = ml.x == -INFINITY ? 0.f : exp2f(ml.x - M);
        float sum = ml.y * w;  // (l is 0 there, or NaN from scores of NaN, which must come through)
#pragma unroll
        for (int s = 16; s > 0; s >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, s);
        L = fmaf(L, keep, sum);
#pragma unroll
        for (int v = 0; v < kV; ++v) acc[v] = make_float2(acc[v].x * keep, acc[v].y * keep);
        uint32_t k = 0;
#pragma unroll 1
        do {
            float2 x[kAhead][kV];
            float wa[kAhead];
#pragma unroll
            for (uint32_t a = 0; a < kAhead; ++a) {
                const uint64_t at = __shfl_sync(0xffffffffu, reinterpret_cast<uint64_t>(o), (k + a) & 31u);
                wa[a] = __shfl_sync(0xffffffffu, w, (k + a) & 31u);
#pragma unroll
                for (int v = 0; v < kV; ++v) {
                    x[a][v] = make_float2(0.f, 0.f);
                    if (k + a < here) x[a][v] = __ldcg(reinterpret_cast<const float2*>(at) + lane + 32 * v);
                }
            }
#pragma unroll
            for (uint32_t a = 0; a < kAhead; ++a) {
                if (wa[a] == 0.f) continue;  // (NaN from a piece that weighs nothing stays out)
#pragma unroll
                for (int v = 0; v < kV; ++v) {
                    acc[v].x = fmaf(x[a][v].x, wa[a], acc[v].x);
                    acc[v].y = fmaf(x[a][v].y, wa[a], acc[v].y);
                }
            }
            k += kAhead;
        } while (k < here);
        if (warm != 0) {
            base += 32;
        } else {
            warm = 1;
            pdl_wait();
            M = -INFINITY;
            L = 0.f;
#pragma unroll
            for (int v = 0; v < kV; ++v) acc[v] = make_float2(0.f, 0.f);
        }
    } while (base < n);
    const float inv = 1.f / L;
#pragma unroll
    for (int v = 0; v < kV; ++v) out[lane + 32 * v] = make_float2(acc[v].x * inv, acc[v].y * inv);
}

// How a call is cut into pieces, from host-side facts alone (the workspace
// size and the launches must agree on it).
struct Plan {
    PrefixGroups groups;
    bool direct;               // one launch, each row reading all of its pages
    uint32_t grid;             // prefix CTAs (0: nothing shared)
    bool fused;                // the tail's CTAs write O
    bool stream;               // no group has more than one tile of query rows
    uint32_t pages_per_split;  // tail splits
    uint32_t max_splits;       // 0: no row has pages of its own
    uint64_t off_ml, off_tail, bytes;
};

bool fast_shape(const CacheView& c, uint32_t q_heads) {
    return (c.dtype == KVFX_BF16 || c.dtype == KVFX_F16) && c.bs == 16 && (c.hd == 64 || c.hd == 128) &&
           c.num_blocks * c.heads < (1ull << 30) && q_heads <= 65535;
}

bool make_plan(const CacheView& c, const kvfx_prefix_group* groups, uint32_t n, uint32_t q_heads, uint64_t max_len,
               Plan* plan) {
    if (!fast_shape(c, q_heads)) return false;
    const uint64_t q_group = q_heads / c.heads, max_pages = ceil_div(max_len, 16);
    if (max_pages >= (1ull << 31)) return false;
    PrefixGroups& gs = plan->groups;
    plan->stream = true;
    gs.n = n;
    uint64_t rows = 0, pairs = 0, tiles = 0, tail_pages = 0, longest = 0;
    for (uint32_t g = 0; g < n; ++g) {
        const uint64_t pages = groups[g].prefix_tokens / 16;
        const uint64_t group_pairs = pages != 0 ? c.heads * ceil_div(groups[g].rows * q_group, 128) : 0;
        rows += groups[g].rows;
        longest = std::max(longest, pages);
        pairs += group_pairs;
        if (group_pairs > c.heads) plan->stream = false;
        tiles += group_pairs * ceil_div(pages, 8);
        if (tiles >= (1ull << 31)) return false;
        tail_pages = std::max(tail_pages, max_pages - pages);
        gs.row_end[g] = static_cast<uint32_t>(rows);
        gs.pages[g] = static_cast<uint32_t>(pages);
        gs.pair_end[g] = static_cast<uint32_t>(pairs);
        gs.tile_end[g] = static_cast<uint32_t>(tiles);
    }
    // Short rows: one launch, in which every row reads all of its pages (the
    // shared ones from the L2), ends before three that share them. B200, us
    // in a graph, 4 rows x 8 heads: 5.9 against 10.0 at 144 tokens, 7.5 / 10.0
    // at 272, 10.5 / 10.2 at 528 (where the two launches saved on the host
    // decide), 16.5 / 11.2 at 1040; as long as one wave of CTAs holds them
    // (64 rows x 32 heads: 16.3 / 16.2 at 272, 23.4 / 17.5 at 528).
    plan->direct = max_pages <= 40 && rows * c.heads * ceil_div(q_group, 8) <=
                                          3 * static_cast<uint64_t>(device_sm_count(c.device));
    if (plan->direct) {
        plan->fused = false;
        plan->grid = 0;
        plan->pages_per_split = decode_tail_split(c, max_pages, static_cast<uint32_t>(max_pages));
        plan->max_splits = 1;
        plan->off_ml = plan->off_tail = plan->bytes = 0;
        return true;
    }
    // One CTA per SM; more where a run would pass the 256 tiles one CTA lists.
    plan->grid = static_cast<uint32_t>(
        umin64(tiles, std::max<uint64_t>(device_sm_count(c.device), ceil_div(tiles, 256))));
    plan->pages_per_split = 1;
    plan->max_splits = 0;
    if (tail_pages != 0) {
        // One split a row, whose CTA joins the prefix's pieces itself (no
        // merge kernel), where it is short or the rows fill the GPU anyway:
        // 256 rows x 64 heads behind 16384 tokens 385 us against 410 with the
        // merge kernel, 64 rows x 32 heads behind 8 prompts 62 / 64. Few rows
        // of some length are better split (16 rows x 8 KV heads of up to 32
        // pages: 18.5 fused, 16.5 split). The bound is the host's (the longest
        // row less the shortest prefix), so rows of 64 pages can stand at its
        // end, as those of the 8 prompts do. Rows that all are as long as it
        // says, behind 4096 tokens, fused / split, at 64, 256, 512 and 1024
        // pages: 40 rows x 8 KV heads 43 / 47, 117 / 117, 219 / 213 and 422 /
        // 403 us; 64 rows 69 / 62, 205 / 175, 385 / 328 and 748 / 620 (512
        // CTAs, a wave of 444 and a rest as long as the wave); 48 rows x 8 KV
        // heads of 64 dims 46 / 54 at 128 pages, 132 / 142 at 512; 256 rows
        // 1222 / 1233 at 512.
        const uint64_t ctas = rows * c.heads * ceil_div(q_group, 8);
        uint32_t pps = decode_pages_per_split(c, rows, q_heads, tail_pages * 16, 0);
        if (tail_pages <= 16 || (tail_pages <= 512 && ctas >= 2 * static_cast<uint64_t>(device_sm_count(c.device)))) {
            pps = static_cast<uint32_t>(tail_pages);
        }
        plan->pages_per_split = decode_tail_split(c, tail_pages, pps);
        plan->max_splits = static_cast<uint32_t>(ceil_div(tail_pages, plan->pages_per_split));
    }
    // A fused CTA keeps at most 256 segments' weights. A prefix of 2^18 pages
    // has 2^15 tiles, which lie in at most 148 runs, or, where there are more
    // CTAs, in runs of 254 to 256 tiles: at most 131 of them.
    plan->fused = plan->max_splits == 1 && longest <= 1u << 18;
    const uint64_t slots = plan->grid != 0 ? plan->grid + pairs : 0;
    auto align = [](uint64_t b) { return (b + 255) & ~uint64_t(255); };
    plan->off_ml = align(slots * 128 * c.hd * 4);
    plan->off_tail = plan->off_ml + align(slots * 128 * 8);
    plan->bytes = plan->off_tail +
                  (plan->fused ? 0 : align(rows * c.heads * ceil_div(q_group, 8) * plan->max_splits * 8 * (c.hd + 2) * 4));
    return true;
}

template <int HD>
cudaError_t launch_merge(const MergeParams& p, uint32_t rows, cudaStream_t s) {
    const uint64_t items = static_cast<uint64_t>(rows) * p.q_heads;
    return launch_dependent(merge_kernel<HD>, dim3(static_cast<uint32_t>(ceil_div(items, kMergeWarps))),
                            dim3(kMergeWarps * 32), s, p);
}

}  // namespace

uint64_t shared_workspace_bytes(const CacheView& c, const kvfx_prefix_group* groups, uint32_t num_groups,
                                uint32_t q_heads, uint64_t max_len) {
    Plan plan;
    return make_plan(c, groups, num_groups, q_heads, max_len, &plan) ? plan.bytes : 0;
}

cudaError_t launch_decode_shared(const CacheView& c, const SharedArgs& a, unsigned* status, cudaStream_t s) {
    Plan plan;
    const bool aligned = ((reinterpret_cast<uintptr_t>(a.q) | reinterpret_cast<uintptr_t>(a.o) |
                           reinterpret_cast<uintptr_t>(c.k) | reinterpret_cast<uintptr_t>(c.v)) & 15u) == 0;
    if (!make_plan(c, a.groups, a.num_groups, a.q_heads, a.max_len, &plan) || !aligned) {
        // Row by row, each reading all of its pages, shared ones too, one warp
        // a query head: 16 rows of 32 + 8 FP32 heads of 128 behind 2064 tokens
        // 1.2 ms.
        uint64_t rows = 0;
        for (uint32_t g = 0; g < a.num_groups; ++g) rows += a.groups[g].rows;
        GenericAttnArgs g{a.q, a.o, a.table, a.max_blocks, a.lens, rows, 0, a.q_heads};
        g.groups = a.groups;
        g.num_groups = a.num_groups;
        g.max_len = a.max_len;
        return launch_attention_generic(c, g, status, s);
    }
    cudaError_t err = cudaSuccess;
    const CacheMaps* maps = cache_maps(c, &err);
    if (maps == nullptr) return err != cudaSuccess ? err : cudaErrorInvalidValue;
    char* ws = static_cast<char*>(a.workspace);
    float* part_o = reinterpret_cast<float*>(ws);
    float* part_ml = reinterpret_cast<float*>(ws + plan.off_ml);
    float* tail = reinterpret_cast<float*>(ws + plan.off_tail);
    if (plan.grid != 0) {
        const PrefixArgs pa{a.q, a.table, a.max_blocks, a.q_heads, plan.grid, plan.stream, &plan.groups, part_o, part_ml,
                            a.lose_prefix};
        const CacheMaps* groups = prefix_maps(c, &err);
        if (groups == nullptr) return err != cudaSuccess ? err : cudaErrorInvalidValue;
        err = launch_prefix_tc(c, pa, *groups, status, s);
        if (err != cudaSuccess) return err;
    }
    const uint32_t tiles = plan.groups.tiles();
    const uint64_t tiles_inv = tiles > 1 ? ~0ull / tiles + (~0ull % tiles == tiles - 1 ? 1 : 0) : ~0ull;
    const PrefixPieces pieces{part_o, part_ml, tiles_inv, plan.grid};
    if (plan.max_splits != 0) {
        const TailArgs ta{a.q, a.o, a.table, a.lens, a.max_blocks, a.max_len, a.q_heads, plan.pages_per_split,
                          plan.max_splits, &plan.groups, tail, pieces, plan.grid != 0, plan.fused, plan.direct};
        err = launch_decode_tail(c, ta, *maps, status, s);
        if (err != cudaSuccess || plan.direct || plan.fused) return err;
    }
    MergeParams m;
    m.groups = plan.groups;
    m.lens = a.lens;
    m.o = a.o;
    m.pieces = pieces;
    m.tail = tail;
    m.max_len = a.max_len;
    m.max_blocks = a.max_blocks;
    m.q_heads = a.q_heads;
    m.kv_heads = c.heads;
    m.q_group = a.q_heads / c.heads;
    m.chunks = (m.q_group + 7) / 8;
    m.pages_per_split = plan.pages_per_split;
    m.max_splits = plan.max_splits;
    m.status = status;
    const uint32_t rows = plan.groups.rows();
    return c.hd == 128 ? launch_merge<128>(m, rows, s) : launch_merge<64>(m, rows, s);
}

}  // namespace kvfx
