// Attention of a batch's rows over the prefixes they share, on the
// 5th-generation tensor cores: the first kernel of kvfx_decode_shared.
//
// The query heads of one KV head of all rows of a group form a matrix of
// rows x q_group query rows (row-major in the batch row), cut into tiles of
// 128. A pair (KV head, query tile) attends over the group's prefix in KV
// tiles of 128 tokens (8 pages):
//     S = Q K^T, m = rowmax(S), P = 2^(S - m), l = rowsum(P), O = P V
// in base 2 (Q pre-scaled by log2(e) / sqrt(hd)), so a page of the prefix is
// read once per 128 query rows instead of once per row. All pairs' tiles form
// one list that the CTAs share in equal consecutive runs; a run's part of a
// pair (a segment) leaves m, l and the unnormalised O in the workspace, and
// the merge kernel of shared.cu joins them. There is no causal mask: the
// prefix lies before every row's query.
//
// Warp roles (12 warps), one CTA per SM:
//   warp 0, 2   K and V producers: per tile up to 8 pages, one tensor load
//               each (128-byte swizzle, no multicast), into rings of 2 (hd
//               128) or 5 (hd 64) tiles. A load brings a page's 16 rows of one
//               head as [2 groups of 8 rows][hd / 64][8 rows][128 bytes]. The
//               loads' coordinates are worked out ahead by all lanes, so that
//               the issuing lane spends 0.3 us a tile: the rings being short,
//               that time is part of a tile's (1.75 us with 1.5 us of it, 1.45
//               now).
//   warp 1      owns TMEM and issues S(t) = Q K_t^T, Q from TMEM, once PV(t - 2)
//               has read P(t - 2), which lies in the same columns.
//   warp 3      issues O += P(t) V_t, P from TMEM. (One warp issuing both
//               groups in turn spends 0.6 us of a tile's time between them.)
//   warps 4-7   softmax, one query row per thread (TMEM lane = row): row
//               maximum, then P = 2^(S - m) over its own S columns as packed
//               hi/lo pairs.
//   warps 8-11  Q staging and O: every kFlush tiles, and at a segment's end,
//               they add O from TMEM to a sum in shared memory (PV starts
//               from zero again), and store a finished segment's sum.
// Warps all of whose query rows lie past the tile's last one only signal.
// TMEM columns: S/P buffers 0 and 128; O 256; Q behind it (hi then lo halves).
// Precision: Q and P are fed as two 16-bit operands each, hi = round(x) and
// lo = round(x - hi): in bf16 off by at most 2^-17 of x (one bf16 operand alone
// is off by up to 2^-8 of each weight), in fp16 by 2^-23 with an absolute floor
// of 2^-25, which is why P enters times 2^7 there (kWeightShift). The tensor
// cores truncate each sum into the FP32 accumulator, a bias that grows with the
// number of additions (measured over 110 tiles in one accumulator: 2.4e-5 of
// O), hence the sum over flushes, which rounds. (Kept in registers it is code
// that runs out of a cold instruction cache at every segment's end, 6 us more
// at 7 tiles a CTA; left to the merge kernel, 16 tiles a piece, it is 60 MB
// more to write and read at 256 rows x 64 heads.) A flush takes all of O into
// registers and lets the next PV go before it adds: 208 us against 218 at 256
// rows x 64 heads x 16384 tokens, 620 -> 660 TFLOP/s of attention (twice that
// executed), where a tile is bounded by its chain: softmax 1.2 us, PV and QK
// 0.6 us each. O is rescaled in TMEM only when a tile's row maximum passes the
// running one by more than 8.
#include <algorithm>
#include <atomic>
#include <cmath>
#include <type_traits>

#include "common.cuh"
#include "launch.h"
#include "tcgen05.cuh"

namespace kvfx {
namespace {

constexpr int kBM = 128;       // query rows per pair
constexpr int kBN = 128;       // tokens per KV tile
constexpr int kTilePages = kBN / 16;
constexpr int kThreads = 384;  // 12 warps
constexpr int kSBufs = 2;
constexpr uint32_t kTmemCols = 512;
constexpr uint32_t kFlush = 8;     // tiles that PV accumulates in TMEM
constexpr uint32_t kMaxRun = 256;  // tiles, and so segments, of a CTA's run
static_assert(kMaxRun <= kThreads, "a thread per tile lists the segments");
constexpr uint32_t kTmemO = kSBufs * kBN;

template <int HD>
struct Shape {
    static constexpr uint32_t kGroup = 8 * HD * 2;             // 8 rows: hd / 64 swizzled blocks of 1 KiB
    static constexpr uint32_t kPage = 2 * kGroup;              // one page's rows of one head
    static constexpr uint32_t kTile = kTilePages * kPage;      // one K or V tile
    static constexpr int kStages = HD == 128 ? 2 : 5;          // tiles per ring
    static constexpr uint32_t kOffV = kStages * kTile;
    static constexpr uint32_t kOffSum = 2 * kStages * kTile;   // O's sum: [hd / 32][128 rows][32], swizzled
    static constexpr uint32_t kOffQ = kOffSum + kBM * HD * 4;  // 4 KiB a warp: Q on its way in
    static constexpr uint32_t kSmem = kOffQ + 4 * 4096 + 1024;  // + alignment slack
    static constexpr uint32_t kTmemQ = kTmemO + HD;            // hi pairs, then lo pairs (HD / 2 columns each)
    static_assert(kTmemQ + HD <= kTmemCols, "TMEM budget");
};

struct PrefixParams {
    PrefixGroups groups;
    const float* q;
    const uint64_t* table;
    uint64_t max_blocks, num_blocks;
    uint32_t kv_heads, q_group;
    uint32_t stream;   // every page is read by one pair only
    float qscale;
    float* part_o;
    float* part_ml;
    unsigned* status;
};

// A segment: tiles [j, j_end) of one pair, in one CTA's run.
struct __align__(16) Segment {
    uint32_t row0;    // the group's first batch row
    uint32_t m0;      // first query row of the tile in the group's matrix
    uint32_t kh, pages;
    uint32_t j, j_end, slot;
    uint32_t m_rows;  // query rows of this pair's tile (1..128)
};
static_assert(sizeof(Segment) == 32, "two 16-byte reads");

// The segments of this CTA's run, in order, written by all threads (one tile
// of the run each) from the launch's parameters alone, so that the work
// overlaps the kernel ahead and each role only reads its way through the list.
// Returns their number after a __syncthreads of the caller's own.
__device__ __forceinline__ void list_segments(const PrefixParams& p, Segment* list, uint32_t* warp_count) {
    const PrefixGroups& gs = p.groups;
    const uint32_t tid = threadIdx.x, lane = tid & 31u, warp = tid >> 5;
    const uint64_t tiles = gs.tiles();
    const uint32_t begin = static_cast<uint32_t>(tiles * blockIdx.x / gridDim.x);
    const uint32_t end = static_cast<uint32_t>(tiles * (blockIdx.x + 1) / gridDim.x);
    const uint32_t tile = begin + tid;
    Segment s{};
    bool starts = false;
    if (tile < end) {
        const uint32_t g = gs.of_tile(tile);
        const uint32_t tile0 = g == 0 ? 0 : gs.tile_end[g - 1], pair0 = g == 0 ? 0 : gs.pair_end[g - 1];
        s.row0 = g == 0 ? 0 : gs.row_end[g - 1];
        s.pages = gs.pages[g];
        const uint32_t ntiles = (s.pages + kTilePages - 1) / kTilePages;
        const uint32_t pair = (tile - tile0) / ntiles;
        s.j = tile - tile0 - pair * ntiles;
        s.j_end = min(ntiles, s.j + (end - tile));
        const uint32_t rows = (gs.row_end[g] - s.row0) * p.q_group;
        const uint32_t m_tiles = (rows + kBM - 1) / kBM;
        s.kh = pair / m_tiles;
        s.m0 = (pair - s.kh * m_tiles) * kBM;
        s.m_rows = min(static_cast<uint32_t>(kBM), rows - s.m0);
        s.slot = blockIdx.x + pair0 + pair;
        starts = tid == 0 || s.j == 0;
    }
    const uint32_t votes = __ballot_sync(0xffffffffu, starts);
    if (lane == 0) warp_count[warp] = __popc(votes);
    __syncthreads();
    uint32_t at = __popc(votes & ((1u << lane) - 1));
    for (uint32_t w = 0; w < warp; ++w) at += warp_count[w];
    if (starts) list[at] = s;
}

// The pieces of segments whose O never came (a bounded wait ran out): no
// weight, and a sum that makes the rows joined with them NaN, whatever an
// earlier call left in the workspace. Thread r of 128 writes query row r.
// (Inlined behind the loop that it follows: as a call it makes 16 rows behind
// 2064 tokens 16.4 us instead of 16.2.)
__device__ __forceinline__ void lose_segments(const PrefixParams& p, const Segment* list, uint32_t k, uint32_t n,
                                              uint32_t r) {
#pragma unroll 1
    for (; k < n; ++k) {
        if (r < list[k].m_rows) {
            reinterpret_cast<float2*>(p.part_ml)[static_cast<uint64_t>(list[k].slot) * kBM + r] =
                make_float2(-INFINITY, __int_as_float(0x7fc00000));
        }
    }
}

// Walks the list tile by tile: segment k, tile j of its pair, and the running
// tile ordinal t that indexes rings and barriers.
struct Cursor {
    const Segment* list;
    uint32_t n, k, j, j_begin, j_end, pages, t;
    __device__ __forceinline__ Cursor(const Segment* l, uint32_t count) : list(l), n(count), k(0), t(0) { open(); }
    __device__ __forceinline__ void open() {
        if (k < n) {
            j = j_begin = list[k].j;
            j_end = list[k].j_end;
            pages = list[k].pages;
        }
    }
    __device__ __forceinline__ bool valid() const { return k < n; }
    __device__ __forceinline__ bool first() const { return j == j_begin; }
    __device__ __forceinline__ bool last() const { return j + 1 == j_end; }
    __device__ __forceinline__ void step() {
        ++t;
        if (++j < j_end) return;
        ++k;
        open();
    }
    // Pages of tile j (8, fewer in a prefix's last tile).
    __device__ __forceinline__ uint32_t tile_pages() const {
        return min(static_cast<uint32_t>(kTilePages), pages - j * kTilePages);
    }
};

// Producer loop of one ring (K or V), run by a whole warp: tile t goes to slot
// t % stages once the MMA that read tile t - stages has completed (freed[slot],
// one commit per tile). At the end, waits for its own copies in flight.
template <int HD>
__device__ __noinline__ void produce(const PrefixParams& p, const CUtensorMap* map, Cursor c, unsigned char* ring,
                                     uint64_t* full, uint64_t* freed) {
    using S = Shape<HD>;
    const uint32_t lane = threadIdx.x & 31u;
    const bool leader = elect_one();
    auto wait = [&](uint64_t* bar, uint32_t phase) {
        return __all_sync(0xffffffffu, mbar_wait_lean(bar, phase, p.status)) != 0;
    };
    pdl_wait();
    // Where the pages are (in groups of 8 rows, counted through the cache's
    // pages and heads), four tiles (32 pages, one a lane) at a time and the
    // next four fetched behind them, so that a table read's latency is never
    // waited for but at a segment's start.
    const uint64_t* row = nullptr;
    uint32_t pages = 0, kh = 0;
    auto fetch = [&](uint32_t page0) -> uint64_t { return page0 + lane < pages ? __ldg(row + page0 + lane) : 0; };
    auto place = [&](uint64_t id) -> int {
        if (id >= p.num_blocks) {
            raise_flag(p.status, KVFX_FLAG_BAD_INDEX);
            id = 0;
        }
        return static_cast<int>((id * p.kv_heads + kh) * 2);
    };
    // Streamed through the L2, but for groups of several query tiles, which
    // read each page once a tile.
    const uint64_t policy = p.stream ? l2_evict_first() : l2_evict_normal();
    int at = 0;
    uint64_t ids_next = 0;
    uint32_t issued = 0;
    for (; c.valid(); c.step()) {
        if (c.first()) {
            row = p.table + static_cast<uint64_t>(c.list[c.k].row0) * p.max_blocks;
            pages = c.pages;
            kh = c.list[c.k].kh;
            at = place(fetch(c.j / 4 * 32));
            ids_next = fetch(c.j / 4 * 32 + 32);
        } else if (c.j % 4 == 0) {
            at = place(ids_next);
            ids_next = fetch((c.j / 4 + 1) * 32);
        }
        int tile_at[kTilePages];
#pragma unroll
        for (int pg = 0; pg < kTilePages; ++pg) tile_at[pg] = __shfl_sync(0xffffffffu, at, c.j % 4 * 8 + pg);
        const uint32_t st = c.t % S::kStages;
        if (c.t >= S::kStages && !wait(&freed[st], (c.t / S::kStages - 1) & 1u)) break;
        const uint32_t n = c.tile_pages();
        if (leader) {
            mbar_arrive_expect_tx(&full[st], n * S::kPage);
#pragma unroll
            for (uint32_t pg = 0; pg < kTilePages; ++pg) {
                if (pg < n)
                    tma_load_4d_hint(ring + st * S::kTile + pg * S::kPage, map, 0, 0, 0, tile_at[pg], &full[st], policy);
            }
        }
        issued = c.t + 1;
    }
    for (uint32_t t = issued > S::kStages ? issued - S::kStages : 0; t < issued; ++t)
        (void)wait(&full[t % S::kStages], (t / S::kStages) & 1u);
}

template <int HD, typename T>
__global__ void __launch_bounds__(kThreads, 1)
prefix_tc_kernel(const __grid_constant__ PrefixParams p, const __grid_constant__ CUtensorMap kmap,
                 const __grid_constant__ CUtensorMap vmap) {
    using S = Shape<HD>;
    extern __shared__ unsigned char smem_raw[];
    __shared__ uint64_t k_full[S::kStages], k_free[S::kStages], v_full[S::kStages], v_free[S::kStages];
    __shared__ uint64_t s_full[kSBufs], p_full[kSBufs], pv_done[kSBufs];
    __shared__ uint64_t q_full, q_free, o_full, o_free, mma_done;
    __shared__ uint64_t ml_full[2], ml_free[2];
    __shared__ float2 ml_sh[2][kBM];  // row maxima and sums at a flush, by flush parity
    __shared__ uint32_t tmem_base_slot, warp_count[kThreads / 32];
    __shared__ Segment list[kMaxRun];

    unsigned char* smem = reinterpret_cast<unsigned char*>(
        (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    const uint32_t sbase = smem_addr(smem);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

    if (tid == 0) {
        for (int s = 0; s < S::kStages; ++s) {
            mbar_init(&k_full[s], 1);
            mbar_init(&k_free[s], 1);
            mbar_init(&v_full[s], 1);
            mbar_init(&v_free[s], 1);
        }
        for (int b = 0; b < kSBufs; ++b) {
            mbar_init(&s_full[b], 1);
            mbar_init(&p_full[b], 128);
            mbar_init(&pv_done[b], 1);
        }
        mbar_init(&q_full, 128);
        mbar_init(&q_free, 1);
        mbar_init(&o_full, 1);
        mbar_init(&o_free, 128);
        for (int b = 0; b < 2; ++b) {
            mbar_init(&ml_full[b], 128);
            mbar_init(&ml_free[b], 128);
        }
        mbar_init(&mma_done, 2);
        fence_mbarrier_init();
    }
    if (warp == 0 && elect_one()) prefetch_tensormap(&kmap);
    if (warp == 2 && elect_one()) prefetch_tensormap(&vmap);
    if (warp == 1) {
        tc::tmem_alloc(&tmem_base_slot, kTmemCols);
        tc::tmem_relinquish();
    }
    list_segments(p, list, warp_count);
    tc::fence_before_sync();
    __syncthreads();
    tc::fence_after_sync();
    const uint32_t tmem = tmem_base_slot;
    uint32_t n_seg = 0;
    for (int w = 0; w < kThreads / 32; ++w) n_seg += warp_count[w];
    const Cursor start(list, n_seg);

    // Each role that reads or writes memory waits for the kernel ahead just
    // before it does.
    if (warp == 0) {
        produce<HD>(p, &kmap, start, smem, k_full, k_free);
    } else if (warp == 2) {
        produce<HD>(p, &vmap, start, smem + S::kOffV, v_full, v_free);
    } else if (warp == 1) {
        // ------------------------------------------------------ QK issuer ---
        // The whole warp runs the schedule; one elected lane issues.
        const bool leader = elect_one();
        auto wait = [&](uint64_t* bar, uint32_t phase) {
            return __all_sync(0xffffffffu, mbar_wait_lean(bar, phase, p.status)) != 0;
        };
        const uint32_t id_qk = tc::idesc_f16(kBM, kBN, std::is_same<T, __nv_bfloat16>::value, false);
        // K: 8-token groups kGroup apart, 64 dims to the next block 1 KiB.
        const uint64_t k_desc0 = tc::smem_desc(sbase, 16, S::kGroup);
        // S(t) = Q K_t^T into S[t % 2], once PV(t - 2) has read P(t - 2) there.
        for (Cursor c = start; c.valid(); c.step()) {
            const uint32_t st = c.t % S::kStages, b = c.t % kSBufs;
            if (c.first() && !wait(&q_full, c.k & 1u)) break;
            if (!wait(&k_full[st], (c.t / S::kStages) & 1u)) break;
            if (c.t >= kSBufs && !wait(&pv_done[b], (c.t / kSBufs - 1) & 1u)) break;
            tc::fence_after_sync();
            const uint32_t d = tmem + b * kBN;
            const uint64_t k_desc = k_desc0 + ((st * S::kTile) >> 4);
            if (leader) {
                // Q_hi, then Q_lo, in K-steps of 16 dims (8 columns of Q; 64
                // dims to a 1 KiB block of K).
#pragma unroll
                for (uint32_t i = 0; i < HD / 8; ++i) {
                    const uint32_t kk = i % (HD / 16);
                    tc::mma_ts(d, tmem + S::kTmemQ + i * 8, k_desc + (((kk >> 2) * 1024 + (kk & 3) * 32) >> 4), id_qk,
                               i > 0 ? 1u : 0u);
                }
                tc::commit(&s_full[b]);
                tc::commit(&k_free[st]);
                if (c.last()) tc::commit(&q_free);  // Q may be replaced once this completes
            }
        }
        // Every MMA issued is complete before TMEM is released.
        if (leader) tc::commit(&mma_done);
        (void)wait(&mma_done, 0);
    } else if (warp == 3) {
        // ------------------------------------------------------ PV issuer ---
        // First: the next kernel may start once what lies ahead of this one
        // is complete (the tail kernel reads Q, K, V and tables without a wait).
        pdl_wait();
        pdl_allow_next();
        const bool leader = elect_one();
        auto wait = [&](uint64_t* bar, uint32_t phase) {
            return __all_sync(0xffffffffu, mbar_wait_lean(bar, phase, p.status)) != 0;
        };
        const uint32_t id_pv = tc::idesc_f16(kBM, HD, std::is_same<T, __nv_bfloat16>::value, true);
        // V (MN-major): the next 64 dims 1 KiB on, 8-token groups kGroup apart.
        const uint64_t v_desc0 = tc::smem_desc(sbase + S::kOffV, 1024, S::kGroup);
        // O += P(t) V_t over the tile's valid pages (16 tokens = one K-step).
        // A flush's first PV overwrites O, which must have been read.
        uint32_t flush = 0, in_flush = 0;
        for (Cursor c = start; c.valid(); c.step()) {
            const uint32_t st = c.t % S::kStages, b = c.t % kSBufs;
            const bool first = in_flush == 0, last = c.last() || in_flush + 1 == kFlush;
            if (first && flush >= 1 && !wait(&o_free, (flush - 1) & 1u)) break;
            if (!wait(&v_full[st], (c.t / S::kStages) & 1u)) break;
            if (!wait(&p_full[b], (c.t / kSBufs) & 1u)) break;
            tc::fence_after_sync();
            const uint32_t pt = tmem + b * kBN, n = c.tile_pages();
            const uint64_t v_desc = v_desc0 + ((st * S::kTile) >> 4);
            if (leader) {
                // Per page, P_hi then P_lo (chunks of 32 tokens: 16 columns
                // of hi pairs, 16 of lo pairs).
#pragma unroll
                for (uint32_t t = 0; t < kTilePages; ++t) {
                    if (t >= n) break;
                    const uint32_t a = pt + (t >> 1) * 32 + (t & 1) * 8;
                    const uint64_t v = v_desc + ((t * S::kPage) >> 4);
                    tc::mma_ts(tmem + kTmemO, a, v, id_pv, (!first || t > 0) ? 1u : 0u);
                    tc::mma_ts(tmem + kTmemO, a + 16, v, id_pv, 1u);
                }
                tc::commit(&pv_done[b]);
                tc::commit(&v_free[st]);
                if (last) tc::commit(&o_full);
            }
            in_flush = last ? 0 : in_flush + 1;
            flush += last ? 1 : 0;
        }
        if (leader) tc::commit(&mma_done);
        (void)wait(&mma_done, 0);
    } else if (warp >= 4 && warp < 8) {
        // -------------------------------------------------------- softmax ---
        const uint32_t quarter = static_cast<uint32_t>(warp & 3);  // TMEM lanes this warp may access
        const uint32_t r = quarter * 32 + lane;                     // query row within the tile
        const uint32_t lane_base = (quarter * 32) << 16;
        const uint32_t tO = tmem + kTmemO + lane_base;
        // tcgen05.ld/st are warp-collective: every wait result is made
        // warp-uniform so that no lane skips one the others execute.
        auto wait_all = [&](uint64_t* bar, uint32_t phase) {
            return __all_sync(0xffffffffu, mbar_wait_lean(bar, phase, p.status)) != 0;
        };
        Cursor c = start;
        float m_run = -INFINITY, l_run = 0.f;
        uint32_t m_rows = 0, flush = 0, in_flush = 0;
        while (c.valid()) {
            const uint32_t t = c.t, b = t % kSBufs;
            if (!wait_all(&s_full[b], (t / kSBufs) & 1u)) break;
            tc::fence_after_sync();
            const bool end = c.last(), last = end || in_flush + 1 == kFlush;
            if (c.first()) m_rows = c.list[c.k].m_rows;
            if (quarter * 32 < m_rows) {
                const uint32_t tS = tmem + b * kBN + lane_base;
                // Scores of pages past the prefix (its last tile) become -inf
                // whatever they held.
                if (c.tile_pages() < kTilePages) {
                    uint32_t none[16];
#pragma unroll
                    for (int e = 0; e < 16; ++e) none[e] = 0xff800000u;
#pragma unroll 1
                    for (uint32_t pg = c.tile_pages(); pg < kTilePages; ++pg) tc::st16(tS + pg * 16, none);
                    tc::wait_st();
                }
                auto max32 = [](const float* v) {
                    float m[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) m[e] = fmax3(v[e], v[4 + e], v[8 + e]);
#pragma unroll
                    for (int q = 12; q < 28; q += 8) {
#pragma unroll
                        for (int e = 0; e < 4; ++e) m[e] = fmax3(m[e], v[q + e], v[q + 4 + e]);
                    }
#pragma unroll
                    for (int e = 0; e < 4; ++e) m[e] = fmaxf(m[e], v[28 + e]);
                    return fmaxf(fmax3(m[0], m[1], m[2]), m[3]);
                };
                float mx;
                {
                    float sc[kBN];
#pragma unroll
                    for (int cb = 0; cb < kBN; cb += 32) tc::ld32(tS + cb, sc + cb);
                    tc::wait_ld32(sc);
                    tc::reg_fence32(sc + 32);
                    tc::reg_fence32(sc + 64);
                    tc::reg_fence32(sc + 96);
                    mx = fmaxf(fmaxf(max32(sc), max32(sc + 32)), fmaxf(max32(sc + 64), max32(sc + 96)));
                }
                // m_run is the maximum less kWeightShift (-inf: replaced by any
                // finite one). The difference is exact near the bound, where
                // m_run + 15 rounds once scores pass 2^24.
                const bool need = mx - m_run > 8.f + kWeightShift<T>;
                const float m_new = mx - kWeightShift<T>;
                const float alpha = need ? ex2_approx(m_run - m_new) : 1.f;  // 0 at the first tile
                l_run *= alpha;
                if (in_flush != 0 && __any_sync(0xffffffffu, need)) {
                    // O holds the flush's earlier tiles once PV(t - 1)
                    // completes; PV(t) waits for this tile's P.
                    if (!wait_all(&pv_done[(t - 1) % kSBufs], ((t - 1) / kSBufs) & 1u)) break;
                    tc::fence_after_sync();
#pragma unroll 1
                    for (uint32_t cb = 0; cb < HD; cb += 32) {
                        float ov[32];
                        tc::ld32(tO + cb, ov);
                        tc::wait_ld32(ov);
#pragma unroll
                        for (int e = 0; e < 32; ++e) ov[e] *= alpha;
                        tc::st32(tO + cb, ov);
                    }
                }
                if (need) m_run = m_new;
                // P over its own S columns: chunk of 32 tokens -> 16 columns
                // of hi pairs, 16 of lo pairs. The scores are read again
                // chunk by chunk, the next one's load under this one's math.
                const float m_sub = m_run == -INFINITY ? 0.f : m_run;  // no score above -inf yet: weights of 0
                const uint64_t mm = f2_pack(m_sub, m_sub);
                uint64_t sum0 = f2_pack(0.f, 0.f), sum1 = sum0;
                auto p_chunk = [&](int ch, float* v) {
                    uint32_t hi[16], lo[16];
#pragma unroll
                    for (int e = 0; e < 16; ++e) {
                        float x0, x1;
                        f2_unpack(f2_sub(f2_pack(v[2 * e], v[2 * e + 1]), mm), x0, x1);
                        x0 = ex2_approx(x0);
                        x1 = ex2_approx(x1);
                        const uint64_t pe = f2_pack(x0, x1);
                        if (e & 1) sum1 = f2_add(sum1, pe);
                        else sum0 = f2_add(sum0, pe);
                        hi[e] = Elem<T>::pack(x0, x1);
                        float r0, r1;
                        f2_unpack(f2_sub(pe, widen2<T>(hi[e])), r0, r1);
                        lo[e] = Elem<T>::pack(r0, r1);
                    }
                    tc::st16(tS + 32 * ch, hi);
                    tc::st16(tS + 32 * ch + 16, lo);
                };
                {
                    float va[32], vb[32];
                    tc::ld32(tS, va);
                    tc::wait_ld32(va);
#pragma unroll 1
                    for (int ch = 0; ch < kBN / 32; ch += 2) {
                        tc::ld32(tS + 32 * (ch + 1), vb);
                        p_chunk(ch, va);
                        tc::wait_ld32(vb);
                        if (ch + 2 < kBN / 32) tc::ld32(tS + 32 * (ch + 2), va);
                        p_chunk(ch + 1, vb);
                        if (ch + 2 < kBN / 32) tc::wait_ld32(va);
                    }
                }
                float s0, s1, s2, s3;
                f2_unpack(sum0, s0, s1);
                f2_unpack(sum1, s2, s3);
                l_run += (s0 + s1) + (s2 + s3);
                tc::wait_st();
            }
            tc::fence_before_sync();
            mbar_arrive(&p_full[b]);
            if (last) {  // the scale of this flush's O, and the segment's sum so far
                const uint32_t mb = flush & 1u;
                if (flush >= 2 && !wait_all(&ml_free[mb], ((flush - 2) >> 1) & 1u)) break;
                ml_sh[mb][r] = make_float2(m_run, l_run);
                mbar_arrive(&ml_full[mb]);
            }
            in_flush = last ? 0 : in_flush + 1;
            flush += last ? 1 : 0;
            if (end) {
                m_run = -INFINITY;
                l_run = 0.f;
            }
            c.step();
        }
    } else if (warp >= 8) {
        // ---------------------------------------------- Q staging and O ---
        const uint32_t quarter = static_cast<uint32_t>(warp & 3);
        const uint32_t r = quarter * 32 + lane;
        const uint32_t lane_base = (quarter * 32) << 16;
        const uint32_t tO = tmem + kTmemO + lane_base;
        auto wait_all = [&](uint64_t* bar, uint32_t phase) {
            return __all_sync(0xffffffffu, mbar_wait_lean(bar, phase, p.status)) != 0;
        };
        // Rows of 32 floats between registers (thread = row) and memory go
        // through this warp's 4 KiB of shared memory, 16-byte chunks swizzled
        // by row, so that 8 lanes move 128 contiguous bytes of a row (a lane
        // per row would touch 32 lines an instruction).
        float4* q_in = reinterpret_cast<float4*>(smem + S::kOffQ + quarter * 4096);
        float4* sum = reinterpret_cast<float4*>(smem + S::kOffSum + quarter * 4096);  // + 16 KiB per 32 columns
        const uint32_t x_row = lane / 8, x_e = lane & 7u;  // this lane's part of the memory side: rows x_row + 4 i
        // Query rows of segment s, scaled, into the Q columns as hi and lo
        // halves (column c of a half holds dims 2c, 2c + 1). Rows past the
        // last one repeat it: their scores and weights stay in their own TMEM
        // lanes and are not stored.
        auto stage_q = [&](const Segment& s) {
            if (quarter * 32 < s.m_rows) {
                const uint32_t last_row = s.m_rows - 1u;
                const float4* src[8];
#pragma unroll
                for (uint32_t i = 0; i < 8; ++i) {
                    const uint32_t m = s.m0 + min(quarter * 32 + i * 4 + x_row, last_row);
                    const uint32_t row = m / p.q_group;
                    const uint64_t qh = static_cast<uint64_t>(s.row0 + row) * p.kv_heads * p.q_group +
                                        static_cast<uint64_t>(s.kh) * p.q_group + (m - row * p.q_group);
                    src[i] = reinterpret_cast<const float4*>(p.q + qh * HD) + x_e;
                }
                const uint64_t qs2 = f2_pack(p.qscale, p.qscale);
                const uint32_t tQ = tmem + S::kTmemQ + lane_base;
                float4 in[8];
#pragma unroll
                for (uint32_t i = 0; i < 8; ++i) in[i] = __ldg(src[i]);
#pragma unroll 1
                for (uint32_t piece = 0; piece < HD / 32; ++piece) {
#pragma unroll
                    for (uint32_t i = 0; i < 8; ++i) {
                        const uint32_t row = i * 4 + x_row;
                        q_in[row * 8 + (x_e ^ (row & 7u))] = in[i];
                    }
                    __syncwarp();
                    if (piece + 1 < HD / 32) {
#pragma unroll
                        for (uint32_t i = 0; i < 8; ++i) in[i] = __ldg(src[i] + (piece + 1) * 8);
                    }
                    uint32_t hi[16], lo[16];
#pragma unroll
                    for (uint32_t e = 0; e < 8; ++e) {
                        const float4 f = q_in[lane * 8 + (e ^ (lane & 7u))];
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            const uint64_t x = f2_mul(h ? f2_pack(f.z, f.w) : f2_pack(f.x, f.y), qs2);
                            float x0, x1;
                            f2_unpack(x, x0, x1);
                            hi[2 * e + h] = Elem<T>::pack(x0, x1);
                            float r0, r1;
                            f2_unpack(f2_sub(x, widen2<T>(hi[2 * e + h])), r0, r1);
                            lo[2 * e + h] = Elem<T>::pack(r0, r1);
                        }
                    }
                    __syncwarp();
                    tc::st16(tQ + piece * 16, hi);
                    tc::st16(tQ + HD / 2 + piece * 16, lo);
                }
                tc::wait_st();
            }
            tc::fence_before_sync();
            mbar_arrive(&q_full);
        };
        pdl_wait();
        uint32_t flush = 0;
        uint32_t done = 0;
        bool ok = true;
        stage_q(list[0]);
#pragma unroll 1
        for (uint32_t k = 0; k < n_seg; ++k) {
            const uint32_t slot = list[k].slot, m_rows = list[k].m_rows, j_end = list[k].j_end, j0 = list[k].j;
            const bool live = quarter * 32 < m_rows;
            float m_o = -INFINITY, l = 0.f;  // scale of the sum, row sum
#pragma unroll 1
            for (uint32_t j = j0; j < j_end; j += kFlush, ++flush) {
                // The next segment's Q goes up as soon as this one's last QK
                // has read its own, while the last tiles' softmax and PV run.
                if (j + kFlush >= j_end && k + 1 < n_seg) {
                    if (!wait_all(&q_free, k & 1u)) { ok = false; break; }
                    tc::fence_after_sync();
                    stage_q(list[k + 1]);
                }
                const uint32_t mb = flush & 1u;
                if (!wait_all(&ml_full[mb], (flush >> 1) & 1u)) { ok = false; break; }
                const float2 ml = ml_sh[mb][r];
                mbar_arrive(&ml_free[mb]);
                if (!wait_all(&o_full, flush & 1u)) { ok = false; break; }
                tc::fence_after_sync();
                if (live) {
                    // sum = sum 2^(m_o - m) + O; a segment's first flush sets it.
                    const float alpha = m_o == ml.x ? 1.f : ex2_approx(m_o - ml.x);
                    const bool first = j == j0;
                    float v[HD];
#pragma unroll
                    for (uint32_t cb = 0; cb < HD; cb += 32) tc::ld32(tO + cb, v + cb);
                    tc::wait_ld32(v);
#pragma unroll
                    for (uint32_t cb = 32; cb < HD; cb += 32) tc::reg_fence32(v + cb);
                    // O is in registers: the next flush's PV may start.
                    tc::fence_before_sync();
                    mbar_arrive(&o_free);
#pragma unroll
                    for (uint32_t cb = 0; cb < HD; cb += 32) {
                        float4* at = sum + cb * (kBM / 4) + lane * 8;
#pragma unroll
                        for (uint32_t e = 0; e < 8; ++e) {
                            float4 x = make_float4(v[cb + 4 * e], v[cb + 4 * e + 1], v[cb + 4 * e + 2], v[cb + 4 * e + 3]);
                            if (!first) {
                                const float4 y = at[e ^ (lane & 7u)];
                                x = make_float4(fmaf(y.x, alpha, x.x), fmaf(y.y, alpha, x.y), fmaf(y.z, alpha, x.z),
                                                fmaf(y.w, alpha, x.w));
                            }
                            at[e ^ (lane & 7u)] = x;
                        }
                    }
                    m_o = ml.x;
                    l = ml.y;
                } else {
                    tc::fence_before_sync();
                    mbar_arrive(&o_free);
                }
            }
            if (!ok) break;
            ++done;
            if (live) {
                __syncwarp();
                const uint64_t at = static_cast<uint64_t>(slot) * kBM + quarter * 32;
#pragma unroll 1
                for (uint32_t cb = 0; cb < HD; cb += 32) {
#pragma unroll
                    for (uint32_t i = 0; i < 8; ++i) {
                        const uint32_t row = i * 4 + x_row;
                        const float4 x = sum[cb * (kBM / 4) + row * 8 + (x_e ^ (row & 7u))];
                        if (quarter * 32 + row < m_rows)
                            *reinterpret_cast<float4*>(p.part_o + (at + row) * HD + cb + 4 * x_e) = x;
                    }
                }
                if (r < m_rows) reinterpret_cast<float2*>(p.part_ml)[at + lane] = make_float2(m_o, l);
                __syncwarp();
            }
        }
        if (!ok) lose_segments(p, list, done, n_seg, r);
    }

    tc::fence_before_sync();
    __syncthreads();
    if (warp == 1) {
        tc::fence_after_sync();
        tc::tmem_dealloc(tmem, kTmemCols);
    }
}

// In place of the prefix kernel: every segment lost (the self-test's launch).
__global__ void __launch_bounds__(kThreads) lost_prefix_kernel(const __grid_constant__ PrefixParams p) {
    __shared__ uint32_t warp_count[kThreads / 32];
    __shared__ Segment list[kMaxRun];
    list_segments(p, list, warp_count);
    __syncthreads();
    uint32_t n_seg = 0;
    for (int w = 0; w < kThreads / 32; ++w) n_seg += warp_count[w];
    pdl_wait();
    pdl_allow_next();
    if (threadIdx.x < kBM) lose_segments(p, list, 0, n_seg, threadIdx.x);
}

template <int HD, typename T>
cudaError_t launch_hd(const CacheView& c, const PrefixParams& p, uint32_t grid, const CacheMaps& maps,
                      cudaStream_t s) {
    static std::atomic<int> attr_done[64];  // zero-initialised; callers on several threads set the same attribute
    if (c.device < 0 || c.device >= 64 || !attr_done[c.device].load(std::memory_order_acquire)) {
        const cudaError_t e = cudaFuncSetAttribute(prefix_tc_kernel<HD, T>,
                                                   cudaFuncAttributeMaxDynamicSharedMemorySize, Shape<HD>::kSmem);
        if (e != cudaSuccess) return e;
        if (c.device >= 0 && c.device < 64) attr_done[c.device].store(1, std::memory_order_release);
    }
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(grid);
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = Shape<HD>::kSmem;
    cfg.stream = s;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, prefix_tc_kernel<HD, T>, p, maps.k, maps.v);
}

}  // namespace

cudaError_t launch_prefix_tc(const CacheView& c, const PrefixArgs& a, const CacheMaps& maps, unsigned* status,
                             cudaStream_t s) {
    PrefixParams p;
    p.groups = *a.groups;
    p.q = a.q;
    p.table = a.table;
    p.max_blocks = a.max_blocks;
    p.num_blocks = c.num_blocks;
    p.kv_heads = c.heads;
    p.q_group = a.q_heads / c.heads;
    p.stream = a.stream ? 1u : 0u;
    p.qscale = static_cast<float>(1.4426950408889634 / std::sqrt(static_cast<double>(c.hd)));
    p.part_o = a.part_o;
    p.part_ml = a.part_ml;
    p.status = status;
    if (ceil_div(a.groups->tiles(), a.grid) > kMaxRun) return cudaErrorInvalidValue;
    if (a.lose) return launch_dependent(lost_prefix_kernel, dim3(a.grid), dim3(kThreads), s, p);
    if (c.hd == 128) {
        return c.dtype == KVFX_BF16 ? launch_hd<128, __nv_bfloat16>(c, p, a.grid, maps, s)
                                    : launch_hd<128, __half>(c, p, a.grid, maps, s);
    }
    return c.dtype == KVFX_BF16 ? launch_hd<64, __nv_bfloat16>(c, p, a.grid, maps, s)
                                : launch_hd<64, __half>(c, p, a.grid, maps, s);
}

}  // namespace kvfx
