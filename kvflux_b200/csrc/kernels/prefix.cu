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
//   warp 0, 2   K and V producers: per tile up to 8 pages x hd/64 tensor loads
//               (128-byte swizzle, no multicast) into rings of 3 (hd 128) or
//               6 (hd 64) tiles each.
//   warp 1      owns TMEM and issues every tcgen05.mma: S(t) = Q K_t^T with Q
//               from TMEM, two tiles ahead of O += P(t) V_t with P from TMEM.
//   warp 3      idle.
//   warps 4-11  softmax, two threads per query row: warps 4-7 take the first
//               64 tokens of a tile, warps 8-11 the last 64, so that a tile's
//               exponentials take half as long (one thread per row left the
//               tensor pipe waiting); the two agree on the row's maximum
//               through shared memory. The same warps stage Q (each half of
//               the dimensions) and store a finished segment's O. Warps all
//               of whose query rows lie past the tile's last one do nothing
//               but signal.
// TMEM columns: S/P buffers 0 and 128; O 256; Q behind it (hi then lo halves).
// S[t % 2] holds P(t) until PV(t) has read it; QK(t + 2) is issued after PV(t)
// by the same thread, and one thread's MMAs execute in order.
// Precision: Q and P are fed as two 16-bit operands each, hi = round(x) and
// lo = round(x - hi): about 16 mantissa bits (one 16-bit operand alone is off
// by 2^-9 of each weight). O is rescaled only when a tile's row maximum
// passes the running one by more than 8.
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
constexpr uint32_t kTmemO = kSBufs * kBN;

template <int HD>
struct Shape {
    static constexpr int kBoxes = HD / 64;                     // 128-byte swizzle boxes per row
    static constexpr uint32_t kHalf = kBN * 128;               // [128 tokens][64 dims]
    static constexpr uint32_t kTile = kBoxes * kHalf;          // one K or V tile
    static constexpr int kStages = 384 / HD;                   // tiles per ring
    static constexpr uint32_t kOffV = kStages * kTile;
    static constexpr uint32_t kSmem = 2 * kStages * kTile + 1024;  // + alignment slack
    static constexpr uint32_t kTmemQ = kTmemO + HD;            // hi pairs, then lo pairs (HD / 2 columns each)
    static_assert(kTmemQ + HD <= kTmemCols, "TMEM budget");
};

struct PrefixParams {
    PrefixGroups groups;
    const float* q;
    const uint64_t* table;
    uint64_t max_blocks, num_blocks;
    uint32_t kv_heads, q_group;
    float qscale;
    float* part_o;
    float* part_ml;
    unsigned* status;
};

// A segment: tiles [j, j_end) of one pair, in one CTA's run.
struct Segment {
    uint32_t row0;    // the group's first batch row
    uint32_t m_rows;  // query rows of this pair's tile (1..128)
    uint32_t m0;      // first query row of the tile in the group's matrix
    uint32_t kh, pages, j, j_end, slot;
};

// Walks a CTA's run of tiles: segment ordinal k, tile j of its pair, and the
// running tile ordinal t that indexes rings and barriers.
struct Cursor {
    Segment s;
    uint32_t next_tile, run_end, k, t;
    bool valid;
    __device__ __forceinline__ void init(const PrefixParams& p) {
        const uint64_t tiles = p.groups.tiles();
        next_tile = static_cast<uint32_t>(tiles * blockIdx.x / gridDim.x);
        run_end = static_cast<uint32_t>(tiles * (blockIdx.x + 1) / gridDim.x);
        k = t = 0;
        open(p);
    }
    __device__ __forceinline__ void open(const PrefixParams& p) {
        valid = next_tile < run_end;
        if (!valid) return;
        const PrefixGroups& gs = p.groups;
        const uint32_t g = gs.of_tile(next_tile);
        const uint32_t tile0 = g == 0 ? 0 : gs.tile_end[g - 1], pair0 = g == 0 ? 0 : gs.pair_end[g - 1];
        s.row0 = g == 0 ? 0 : gs.row_end[g - 1];
        s.pages = gs.pages[g];
        const uint32_t ntiles = (s.pages + kTilePages - 1) / kTilePages;
        const uint32_t local = next_tile - tile0;
        const uint32_t pair = local / ntiles;
        s.j = local - pair * ntiles;
        s.j_end = min(ntiles, s.j + (run_end - next_tile));
        const uint32_t rows = (gs.row_end[g] - s.row0) * p.q_group;
        const uint32_t m_tiles = (rows + kBM - 1) / kBM;
        s.kh = pair / m_tiles;
        s.m0 = (pair - s.kh * m_tiles) * kBM;
        s.m_rows = min(static_cast<uint32_t>(kBM), rows - s.m0);
        s.slot = blockIdx.x + pair0 + pair;
        next_tile += s.j_end - s.j;
    }
    __device__ __forceinline__ void step(const PrefixParams& p) {
        ++t;
        if (++s.j < s.j_end) return;
        ++k;
        open(p);
    }
    __device__ __forceinline__ bool last() const { return s.j + 1 == s.j_end; }
    // Pages of tile j (8, fewer in a prefix's last tile).
    __device__ __forceinline__ uint32_t tile_pages() const {
        return min(static_cast<uint32_t>(kTilePages), s.pages - s.j * kTilePages);
    }
};

// Producer loop of one ring (K or V), run by a whole warp: tile t goes to slot
// t % stages once the MMA that read tile t - stages has completed (freed[slot],
// one commit per tile). The next tile's page ids are fetched before the wait
// for its slot. At the end, waits for its own copies in flight.
template <int HD>
__device__ __noinline__ void produce(const PrefixParams& p, const CUtensorMap* map, unsigned char* ring,
                                     uint64_t* full, uint64_t* freed) {
    using S = Shape<HD>;
    const uint32_t lane = threadIdx.x & 31u;
    const bool leader = elect_one();
    auto wait = [&](uint64_t* bar, uint32_t phase) {
        return __all_sync(0xffffffffu, mbar_wait_lean(bar, phase, p.status)) != 0;
    };
    if (leader) prefetch_tensormap(map);
    Cursor c;
    c.init(p);
    auto page_id = [&]() -> uint64_t {  // of page `lane` of the cursor's tile
        if (!c.valid || lane >= c.tile_pages()) return 0;
        return __ldg(p.table + static_cast<uint64_t>(c.s.row0) * p.max_blocks + c.s.j * kTilePages + lane);
    };
    uint64_t id = page_id();
    uint32_t issued = 0;
    while (c.valid) {
        const uint32_t st = c.t % S::kStages;
        if (c.t >= S::kStages && !wait(&freed[st], (c.t / S::kStages - 1) & 1u)) break;
        const uint32_t n = c.tile_pages();
        if (leader) mbar_arrive_expect_tx(&full[st], n * S::kBoxes * 2048);
        for (uint32_t pg = 0; pg < n; ++pg) {
            uint64_t blk = __shfl_sync(0xffffffffu, id, pg);
            if (!leader) continue;
            if (blk >= p.num_blocks) {
                raise_flag(p.status, KVFX_FLAG_BAD_INDEX);
                blk = 0;
            }
#pragma unroll
            for (int b = 0; b < S::kBoxes; ++b) {
                tma_load_4d(ring + st * S::kTile + b * S::kHalf + pg * 2048, map, b * 64, 0,
                            static_cast<int>(c.s.kh), static_cast<int>(blk), &full[st]);
            }
        }
        issued = c.t + 1;
        c.step(p);
        id = page_id();
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
    __shared__ uint64_t q_full, o_full, o_free, mma_done;
    __shared__ uint64_t x_full[4][2];       // maxima of a row quarter's two halves exchanged
    __shared__ float x_max[2][2][kBM];      // [exchange parity][half][row]
    __shared__ float l_half[2][kBM];        // [segment parity][row]: second half's row sums
    __shared__ uint64_t l_full[4][2];
    __shared__ uint32_t tmem_base_slot;

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
            mbar_init(&p_full[b], 256);
            mbar_init(&pv_done[b], 1);
        }
        mbar_init(&q_full, 256);
        mbar_init(&o_full, 1);
        mbar_init(&o_free, 256);
        for (int w = 0; w < 4; ++w) {
            for (int b = 0; b < 2; ++b) {
                mbar_init(&x_full[w][b], 64);
                mbar_init(&l_full[w][b], 32);
            }
        }
        mbar_init(&mma_done, 1);
        fence_mbarrier_init();
    }
    if (warp == 1) {
        tc::tmem_alloc(&tmem_base_slot, kTmemCols);
        tc::tmem_relinquish();
    }
    tc::fence_before_sync();
    __syncthreads();
    tc::fence_after_sync();
    const uint32_t tmem = tmem_base_slot;

    // Everything above overlaps the kernel ahead; everything it wrote is
    // complete and visible from here on. Only then may the next kernel start:
    // the tail kernel reads Q, K, V and tables without a wait of its own.
    pdl_wait();
    pdl_allow_next();

    if (warp == 0) {
        produce<HD>(p, &kmap, smem, k_full, k_free);
    } else if (warp == 2) {
        produce<HD>(p, &vmap, smem + S::kOffV, v_full, v_free);
    } else if (warp == 1) {
        // ----------------------------------------------------- MMA issuer ---
        // The whole warp runs the schedule; one elected lane issues.
        const bool leader = elect_one();
        auto wait = [&](uint64_t* bar, uint32_t phase) {
            return __all_sync(0xffffffffu, mbar_wait_lean(bar, phase, p.status)) != 0;
        };
        constexpr bool kBF = std::is_same<T, __nv_bfloat16>::value;
        const uint32_t id_qk = tc::idesc_f16(kBM, kBN, kBF, false);
        const uint32_t id_pv = tc::idesc_f16(kBM, HD, kBF, true);
        const uint64_t k_desc0 = tc::desc_k_major(sbase);
        const uint64_t v_desc0 = tc::desc_mn_major(sbase + S::kOffV, S::kHalf);
        Cursor qk, pv;
        qk.init(p);
        pv.init(p);
        uint32_t qk_seg = 0;  // segments whose Q has been waited for
        // S(t) = Q K_t^T into S[t % 2], whose P(t - 2) PV(t - 2) (issued
        // before by this thread) reads first.
        auto qk_step = [&]() -> bool {
            const uint32_t st = qk.t % S::kStages;
            if (qk.k == qk_seg) {  // a segment's first tile
                if (!wait(&q_full, qk.k & 1u)) return false;
                ++qk_seg;
            }
            if (!wait(&k_full[st], (qk.t / S::kStages) & 1u)) return false;
            tc::fence_after_sync();
            const uint32_t d = tmem + (qk.t % kSBufs) * kBN;
            const uint64_t k_desc = k_desc0 + ((st * S::kTile) >> 4);
            if (leader) {
#pragma unroll
                for (uint32_t i = 0; i < HD / 8; ++i) {  // Q_hi, then Q_lo, in K-steps of 16 dims
                    const uint32_t part = i / (HD / 16), kk = i % (HD / 16);
                    const uint32_t a = tmem + S::kTmemQ + part * (HD / 2) + kk * 8;
                    const uint32_t b_off = (kk >> 2) * S::kHalf + (kk & 3) * 32;
                    tc::mma_ts(d, a, k_desc + (b_off >> 4), id_qk, i > 0 ? 1u : 0u);
                }
                tc::commit(&s_full[qk.t % kSBufs]);
                tc::commit(&k_free[st]);
            }
            qk.step(p);
            return true;
        };
        // O += P(t) V_t over the tile's valid pages (16 tokens = one K-step).
        uint32_t pv_seg = 0;
        auto pv_step = [&]() -> bool {
            const uint32_t st = pv.t % S::kStages, b = pv.t % kSBufs;
            const bool first = pv.k == pv_seg;
            if (first) {  // overwrites O, which the previous segment's epilogue must have read
                if (pv.k >= 1 && !wait(&o_free, (pv.k - 1) & 1u)) return false;
                ++pv_seg;
            }
            if (!wait(&v_full[st], (pv.t / S::kStages) & 1u)) return false;
            if (!wait(&p_full[b], (pv.t / kSBufs) & 1u)) return false;
            tc::fence_after_sync();
            const uint32_t pt = tmem + b * kBN, n = pv.tile_pages();
            const uint64_t v_desc = v_desc0 + ((st * S::kTile) >> 4);
            const bool last = pv.last();
            if (leader) {
#pragma unroll
                for (uint32_t i = 0; i < 2 * kTilePages; ++i) {  // per page, P_hi then P_lo
                    const uint32_t t = i >> 1, part = i & 1;
                    if (t >= n) break;
                    const uint32_t a = pt + (t >> 1) * 32 + part * 16 + (t & 1) * 8;
                    tc::mma_ts(tmem + kTmemO, a, v_desc + ((t * 2048) >> 4), id_pv, (!first || i > 0) ? 1u : 0u);
                }
                tc::commit(&pv_done[b]);
                tc::commit(&v_free[st]);
                if (last) tc::commit(&o_full);
            }
            pv.step(p);
            return true;
        };
        bool ok = true;
        for (int i = 0; i < 2 && ok && qk.valid; ++i) ok = qk_step();
        // PV(t) is committed before QK(t + 2) may wait for its segment's Q,
        // which the softmax warps stage only after tile t + 1 (whose rescale
        // may wait for PV(t)).
        while (ok && pv.valid) {
            ok = pv_step();
            if (ok && qk.valid) ok = qk_step();
        }
        // Every MMA this thread issued is complete before TMEM is released.
        if (leader) tc::commit(&mma_done);
        (void)wait(&mma_done, 0);
    } else if (warp >= 4) {
        // -------------------------- softmax, Q staging, segment epilogue ---
        const uint32_t half = warp >= 8 ? 1u : 0u;
        const uint32_t quarter = static_cast<uint32_t>(warp & 3);  // TMEM lanes this warp may access
        const uint32_t r = quarter * 32 + lane;                     // query row within the tile
        const uint32_t lane_base = (quarter * 32) << 16;
        constexpr uint32_t kQD = HD / 2;                            // dims this thread stages and stores
        const uint32_t d0 = half * kQD;
        const uint32_t tO = tmem + kTmemO + lane_base + d0;
        // tcgen05.ld/st are warp-collective: every wait result is made
        // warp-uniform so that no lane skips one the others execute.
        auto wait_all = [&](uint64_t* bar, uint32_t phase) {
            return __all_sync(0xffffffffu, mbar_wait_lean(bar, phase, p.status)) != 0;
        };
        // Query row r of segment s (its last live row for rows past it: their
        // scores and weights stay in their own TMEM lanes and are not stored).
        auto stage_q = [&](const Segment& s) {
            if (quarter * 32 < s.m_rows) {
                const uint32_t m = s.m0 + min(r, s.m_rows - 1);
                const uint32_t row = m / p.q_group;
                const uint64_t qh = static_cast<uint64_t>(s.row0 + row) * p.kv_heads * p.q_group +
                                    static_cast<uint64_t>(s.kh) * p.q_group + (m - row * p.q_group);
                const float4* src = reinterpret_cast<const float4*>(p.q + qh * HD + d0);
                const uint64_t qs2 = f2_pack(p.qscale, p.qscale);
                const uint32_t tQ = tmem + S::kTmemQ + lane_base + d0 / 2;
                float4 v[kQD / 4];
#pragma unroll
                for (uint32_t e = 0; e < kQD / 4; ++e) v[e] = __ldg(src + e);
#pragma unroll
                for (uint32_t cc = 0; cc < kQD / 16; ++cc) {
                    uint32_t hi[8], lo[8];
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        const float4& f = v[4 * cc + e / 2];
                        const uint64_t x = f2_mul((e & 1) ? f2_pack(f.z, f.w) : f2_pack(f.x, f.y), qs2);
                        float x0, x1;
                        f2_unpack(x, x0, x1);
                        hi[e] = Elem<T>::pack(x0, x1);
                        float r0, r1;
                        f2_unpack(f2_sub(x, widen2<T>(hi[e])), r0, r1);
                        lo[e] = Elem<T>::pack(r0, r1);
                    }
                    tc::st8(tQ + cc * 8, hi);
                    tc::st8(tQ + HD / 2 + cc * 8, lo);
                }
                tc::wait_st();
            }
            tc::fence_before_sync();
            mbar_arrive(&q_full);
        };
        Cursor c;
        c.init(p);
        if (c.valid) stage_q(c.s);
        bool ok = true;
        uint32_t xi = 0;  // exchanges made (both halves of a quarter make the same ones)
        uint32_t li = 0;  // live segments finished, alike
        while (ok && c.valid) {
            const Segment s = c.s;
            const uint32_t seg = c.k;
            const bool live = quarter * 32 < s.m_rows;
            float m_run = -INFINITY, l_run = 0.f;
            // ------------------------------------------------ its tiles ---
            while (c.valid && c.k == seg) {
                const uint32_t t = c.t, b = t % kSBufs;
                if (!wait_all(&s_full[b], (t / kSBufs) & 1u)) { ok = false; break; }
                tc::fence_after_sync();
                if (live) {
                    const uint32_t tS = tmem + b * kBN + lane_base + half * 64;
                    // Columns from `lim` on lie past the prefix (a select, so
                    // that they become -inf whatever they held).
                    const int lim = static_cast<int>(c.tile_pages() * 16) - static_cast<int>(half * 64);
                    float v[64];
                    tc::ld32(tS, v);
                    tc::ld32(tS + 32, v + 32);
                    tc::wait_ld32(v);
                    tc::reg_fence32(v + 32);
                    if (lim < 64) {
#pragma unroll
                        for (int i = 0; i < 64; ++i) v[i] = i < lim ? v[i] : -INFINITY;
                    }
                    float mx;
                    {
                        float m4[4];
#pragma unroll
                        for (int e = 0; e < 4; ++e) m4[e] = fmax3(v[e], v[4 + e], v[8 + e]);
#pragma unroll
                        for (int i = 12; i < 60; i += 8) {
#pragma unroll
                            for (int e = 0; e < 4; ++e) m4[e] = fmax3(m4[e], v[i + e], v[i + 4 + e]);
                        }
#pragma unroll
                        for (int e = 0; e < 4; ++e) m4[e] = fmaxf(m4[e], v[60 + e]);
                        mx = fmaxf(fmax3(m4[0], m4[1], m4[2]), m4[3]);
                    }
                    // The row's maximum over both halves.
                    x_max[xi & 1u][half][r] = mx;
                    mbar_arrive(&x_full[quarter][xi & 1u]);
                    if (!wait_all(&x_full[quarter][xi & 1u], (xi >> 1) & 1u)) { ok = false; break; }
                    mx = fmaxf(mx, x_max[xi & 1u][half ^ 1u][r]);
                    ++xi;
                    const bool need = mx > m_run + 8.f;  // m_run = -inf: at any finite maximum
                    const float alpha = need ? ex2_approx(m_run - mx) : 1.f;  // 0 at the first tile
                    l_run *= alpha;
                    if (c.s.j != s.j && __any_sync(0xffffffffu, need)) {
                        // O holds the segment's earlier tiles once PV(t - 1)
                        // completes; PV(t) waits for this tile's P.
                        if (!wait_all(&pv_done[(t - 1) % kSBufs], ((t - 1) / kSBufs) & 1u)) { ok = false; break; }
                        tc::fence_after_sync();
#pragma unroll 1
                        for (uint32_t cb = 0; cb < kQD; cb += 32) {
                            float ov[32];
                            tc::ld32(tO + cb, ov);
                            tc::wait_ld32(ov);
#pragma unroll
                            for (int e = 0; e < 32; ++e) ov[e] *= alpha;
                            tc::st32(tO + cb, ov);
                        }
                    }
                    if (need) m_run = mx;
                    // P over its own S columns: chunk of 32 tokens -> 16
                    // columns of hi pairs, 16 of lo pairs.
                    const float m_sub = m_run == -INFINITY ? 0.f : m_run;  // no visible score yet: weights of 0
                    const uint64_t mm = f2_pack(m_sub, m_sub);
                    uint64_t sum0 = f2_pack(0.f, 0.f), sum1 = sum0;
#pragma unroll
                    for (int ch = 0; ch < 2; ++ch) {
                        uint32_t hi[16], lo[16];
#pragma unroll
                        for (int e = 0; e < 16; ++e) {
                            float x0, x1;
                            f2_unpack(f2_sub(f2_pack(v[32 * ch + 2 * e], v[32 * ch + 2 * e + 1]), mm), x0, x1);
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
                    }
                    float s0, s1, s2, s3;
                    f2_unpack(sum0, s0, s1);
                    f2_unpack(sum1, s2, s3);
                    l_run += (s0 + s1) + (s2 + s3);
                    tc::wait_st();
                }
                tc::fence_before_sync();
                mbar_arrive(&p_full[b]);
                c.step(p);
            }
            if (!ok) break;
            // The segment's last QK has completed (its S was read above): the
            // next segment's Q goes up while the last PV runs.
            if (c.valid) stage_q(c.s);
            // ------------------------------------------------- epilogue ---
            if (live && half == 1) {
                l_half[li & 1u][r] = l_run;
                mbar_arrive(&l_full[quarter][li & 1u]);
            }
            if (!wait_all(&o_full, seg & 1u)) break;
            tc::fence_after_sync();
            float ov[kQD];
            if (live) {
#pragma unroll
                for (uint32_t cb = 0; cb < kQD; cb += 32) tc::ld32(tO + cb, ov + cb);
                tc::wait_ld32(ov);
                if constexpr (kQD == 64) tc::reg_fence32(ov + 32);
            }
            tc::fence_before_sync();
            mbar_arrive(&o_free);
            if (live) {
                if (r < s.m_rows) {
                    float4* dst = reinterpret_cast<float4*>(p.part_o + (static_cast<uint64_t>(s.slot) * kBM + r) * HD + d0);
#pragma unroll
                    for (uint32_t e = 0; e < kQD / 4; ++e)
                        dst[e] = make_float4(ov[4 * e], ov[4 * e + 1], ov[4 * e + 2], ov[4 * e + 3]);
                }
                if (half == 0) {
                    if (!wait_all(&l_full[quarter][li & 1u], (li >> 1) & 1u)) break;
                    if (r < s.m_rows) {
                        reinterpret_cast<float2*>(p.part_ml)[static_cast<uint64_t>(s.slot) * kBM + r] =
                            make_float2(m_run, l_run + l_half[li & 1u][r]);
                    }
                }
                ++li;
            }
        }
    }

    tc::fence_before_sync();
    __syncthreads();
    if (warp == 1) {
        tc::fence_after_sync();
        tc::tmem_dealloc(tmem, kTmemCols);
    }
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
    p.qscale = static_cast<float>(1.4426950408889634 / std::sqrt(static_cast<double>(c.hd)));
    p.part_o = a.part_o;
    p.part_ml = a.part_ml;
    p.status = status;
    if (c.hd == 128) {
        return c.dtype == KVFX_BF16 ? launch_hd<128, __nv_bfloat16>(c, p, a.grid, maps, s)
                                    : launch_hd<128, __half>(c, p, a.grid, maps, s);
    }
    return c.dtype == KVFX_BF16 ? launch_hd<64, __nv_bfloat16>(c, p, a.grid, maps, s)
                                : launch_hd<64, __half>(c, p, a.grid, maps, s);
}

}  // namespace kvfx
