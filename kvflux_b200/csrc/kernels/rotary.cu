// New tokens' Q, K and V on their way into attention and cache: per-head RMS
// norm of Q and K, rotary position embedding, Q out in FP32 (as the attention
// entry points take it), K and V into their cache slots.
//
//   y_d = x_d / sqrt(mean(x^2) + eps) * w_d          (Q and K; optional)
//   (a, b) -> (a cos - b sin, b cos + a sin)         over rotary_dim dims, the
//       pair being dims (i, i + rotary_dim / 2), or (2i, 2i + 1) interleaved;
//       dims past rotary_dim stay as they are
//   K[slot / bs][h][slot % bs][:] = round(k), V alike unrotated, Q_out = q
//
// Everything is computed in FP32; K is rounded once, to the cache's type.
//
// Bounded by HBM for a prefill chunk (each input read once, each output
// written once) and by memory latency for a decode step. A group of lanes
// holds one head's row, eight elements a lane, and walks the token's heads
// with the token's factors in registers; a pass's rows are loaded while the
// pass before is computed. The norm's sum and the rotation's partner dims
// move by shuffles inside the group. B200, 8192 tokens of 32 + 8 + 8 heads of
// 128 bf16: 49 us, 5.6 TB/s (57 us with 64 threads a CTA, 71 us with 128, 60 us
// without the pass ahead); a decode step's 64 tokens: 3.6 us. In FP32 106 us,
// 3.8 TB/s (spills, see kMinCtas), and 4.4 us.
#include <algorithm>
#include <cmath>

#include "common.cuh"
#include "launch.h"

namespace kvfx {
namespace {

constexpr int kThreads = 32;      // one warp a CTA: many small ones hide the chain of loads a token has
// CTAs per SM: 96 registers. 16-bit rows fit; the four FP32 kernels, whose rows
// in flight are twice as wide, spill 140 to 208 bytes.
constexpr int kMinCtas = 18;
constexpr int kAnyThreads = 128;  // of the element-wise kernel
constexpr int kEl = 8;            // elements per lane
constexpr int kRows = 4;          // rows in flight per lane group, and as many behind them

struct RotatedParams {
    const char* q;
    const char* k;
    const char* v;
    uint64_t q_stride, k_stride, v_stride;  // elements from token to token
    const float* cos_sin;
    const float* q_weight;
    const float* k_weight;
    const uint64_t* positions;
    const uint64_t* slots;
    float* q_out;
    char* k_cache;
    char* v_cache;
    uint64_t max_positions, slot_count;
    uint32_t q_heads, kv_heads, hd, bs, rotary_dim, interleaved;
    float eps, inv_hd;
    unsigned* status;
};

// A lane's eight elements as they are stored.
template <typename T>
struct Raw {
    uint4 w[sizeof(T) / 2];
};

template <typename T>
__device__ __forceinline__ Raw<T> load8(const T* p) {
    Raw<T> r;
#pragma unroll
    for (int i = 0; i < static_cast<int>(sizeof(T) / 2); ++i) r.w[i] = __ldg(reinterpret_cast<const uint4*>(p) + i);
    return r;
}

template <typename T>
__device__ __forceinline__ void store8(T* p, const Raw<T>& r) {
#pragma unroll
    for (int i = 0; i < static_cast<int>(sizeof(T) / 2); ++i) reinterpret_cast<uint4*>(p)[i] = r.w[i];
}

// Pairs (2i, 2i + 1) of the elements as packed floats.
template <typename T>
__device__ __forceinline__ void widen8(const Raw<T>& r, uint64_t (&x)[kEl / 2]) {
    const uint32_t* u = reinterpret_cast<const uint32_t*>(r.w);
#pragma unroll
    for (int i = 0; i < kEl / 2; ++i) {
        if constexpr (sizeof(T) == 2) x[i] = widen2<T>(u[i]);
        else x[i] = f2_pack(__uint_as_float(u[2 * i]), __uint_as_float(u[2 * i + 1]));
    }
}

template <typename T>
__device__ __forceinline__ Raw<T> narrow8(const uint64_t (&x)[kEl / 2]) {
    Raw<T> r;
    uint32_t* u = reinterpret_cast<uint32_t*>(r.w);
#pragma unroll
    for (int i = 0; i < kEl / 2; ++i) {
        float a, b;
        f2_unpack(x[i], a, b);
        if constexpr (sizeof(T) == 2) {
            u[i] = Elem<T>::pack(a, b);
        } else {
            u[2 * i] = __float_as_uint(a);
            u[2 * i + 1] = __float_as_uint(b);
        }
    }
    return r;
}

__device__ __forceinline__ uint64_t f2_swap(uint64_t x) {
    float a, b;
    f2_unpack(x, a, b);
    return f2_pack(b, a);
}

__device__ __forceinline__ void load_f8(const float* p, uint64_t (&x)[kEl / 2]) {
#pragma unroll
    for (int i = 0; i < kEl / 4; ++i) {
        const float4 a = __ldg(reinterpret_cast<const float4*>(p) + i);
        x[2 * i] = f2_pack(a.x, a.y);
        x[2 * i + 1] = f2_pack(a.z, a.w);
    }
}

// 32 contiguous bytes in one store.
__device__ __forceinline__ void store_f8(float* p, const uint64_t (&x)[kEl / 2]) {
    asm volatile("st.global.v4.b64 [%0], {%1, %2, %3, %4};" ::"l"(p), "l"(x[0]), "l"(x[1]), "l"(x[2]), "l"(x[3])
                 : "memory");
}

// Where token t goes: false for a padding token (KVFX_NO_SLOT) and, with the
// bad-index flag, for a slot or position outside the cache or the table.
__device__ __forceinline__ bool token_place(const RotatedParams& p, uint64_t t, uint64_t& pos, uint64_t& slot) {
    pos = __ldg(p.positions + t);
    slot = __ldg(p.slots + t);
    if (slot == KVFX_NO_SLOT) return false;
    if (slot >= p.slot_count || pos >= p.max_positions) {
        raise_flag(p.status, KVFX_FLAG_BAD_INDEX);
        return false;
    }
    return true;
}

// Element offset of head 0's row of a slot in a cache (head h: + h * bs * hd).
__device__ __forceinline__ uint64_t slot_row(const RotatedParams& p, uint64_t slot) {
    const uint64_t page = (p.bs & (p.bs - 1)) == 0 ? slot >> (31 - __clz(static_cast<int>(p.bs))) : slot / p.bs;
    return (page * p.kv_heads * p.bs + (slot - page * p.bs)) * p.hd;
}

// LPR lanes per row (head_size = 8 LPR). One CTA per token and slice of its
// rows (blockIdx.y of gridDim.y); rows are Q heads, K heads, V heads in turn.
// With weight and rotation folded into two factors per dimension, a row is
//     y_d = (x_d a_d + x_partner(d) b_d) / sqrt(mean(x^2) + eps),
// a = w c and b = +- w_partner s, and the partner's x comes as stored (16-bit
// rows: four shuffles a row, and half the instructions of norming first).
// Lanes past rotary_dim take 0 for it: an infinity there stays as it is.
template <typename T, int LPR>
__global__ void __launch_bounds__(kThreads, kMinCtas) write_rotated_kernel(const __grid_constant__ RotatedParams p) {
    constexpr int kGroups = kThreads / LPR;
    constexpr int kHd = LPR * kEl;
    pdl_allow_next();
    pdl_wait();  // launched as a dependent: the previous kernel's writes first
    const uint64_t t = blockIdx.x;
    const int l = threadIdx.x % LPR, g = threadIdx.x / LPR;
    const uint32_t rows = p.q_heads + 2 * p.kv_heads, first_v = p.q_heads + p.kv_heads;
    const uint32_t first = blockIdx.y * kGroups + g, step = gridDim.y * kGroups;
    const int d0 = l * kEl;
    // Shuffles stay inside a row's lanes: the rows of a warp may differ.
    const uint32_t lanes = LPR == 32 ? 0xffffffffu : ((1u << LPR) - 1) << (threadIdx.x & 31 & ~(LPR - 1));

    auto row_ptr = [&](uint32_t r) {
        const T* base = reinterpret_cast<const T*>(p.q) + t * p.q_stride;
        uint32_t h = r;
        if (r >= first_v) {
            base = reinterpret_cast<const T*>(p.v) + t * p.v_stride;
            h = r - first_v;
        } else if (r >= p.q_heads) {
            base = reinterpret_cast<const T*>(p.k) + t * p.k_stride;
            h = r - p.q_heads;
        }
        return base + static_cast<uint64_t>(h) * kHd + d0;
    };
    Raw<T> raw[kRows], next[kRows];
    auto load_rows = [&](uint32_t r0, Raw<T>(&to)[kRows]) {
#pragma unroll
        for (int i = 0; i < kRows; ++i) {
            if (r0 + i * step < rows) to[i] = load8(row_ptr(r0 + i * step));
        }
    };
    load_rows(first, raw);  // independent of the token's place: both latencies overlap
    uint64_t pos, slot;
    if (!token_place(p, t, pos, slot)) return;

    // This lane's factors for Q and for K rows, and where its partner dims are.
    const int rot = static_cast<int>(p.rotary_dim), half = rot / 2;
    uint64_t qa[kEl / 2], qb[kEl / 2], ka[kEl / 2], kb[kEl / 2];
    int partner = l;
    const uint32_t turned = d0 < rot ? ~0u : 0u;
    {
        const float* tab = p.cos_sin + pos * p.rotary_dim;
        uint64_t c[kEl / 2], s[kEl / 2];
#pragma unroll
        for (int i = 0; i < kEl / 2; ++i) {
            c[i] = f2_pack(1.f, 1.f);
            s[i] = 0;
        }
        if (d0 < rot && p.interleaved) {  // pairs (2i, 2i + 1): four angles, partner in the same lane
            const float4 cc = __ldg(reinterpret_cast<const float4*>(tab + d0 / 2));
            const float4 ss = __ldg(reinterpret_cast<const float4*>(tab + half + d0 / 2));
            c[0] = f2_pack(cc.x, cc.x), c[1] = f2_pack(cc.y, cc.y);
            c[2] = f2_pack(cc.z, cc.z), c[3] = f2_pack(cc.w, cc.w);
            s[0] = f2_pack(-ss.x, ss.x), s[1] = f2_pack(-ss.y, ss.y);
            s[2] = f2_pack(-ss.z, ss.z), s[3] = f2_pack(-ss.w, ss.w);
        } else if (d0 < rot) {  // pairs (i, i + rot / 2): the partner lane holds the other half
            const bool low = d0 < half;
            partner = low ? l + half / kEl : l - half / kEl;
            const int a0 = low ? d0 : d0 - half;
            load_f8(tab + a0, c);
            load_f8(tab + half + a0, s);
            const uint64_t sign = low ? f2_pack(-1.f, -1.f) : f2_pack(1.f, 1.f);
#pragma unroll
            for (int i = 0; i < kEl / 2; ++i) s[i] = f2_mul(s[i], sign);
        }
        auto fold = [&](const float* weight, uint64_t (&a)[kEl / 2], uint64_t (&b)[kEl / 2]) {
#pragma unroll
            for (int i = 0; i < kEl / 2; ++i) {
                a[i] = c[i];
                b[i] = s[i];
            }
            if (weight == nullptr) return;
            uint64_t w[kEl / 2], wp[kEl / 2];
            load_f8(weight + d0, w);
            load_f8(weight + partner * kEl, wp);
#pragma unroll
            for (int i = 0; i < kEl / 2; ++i) {
                a[i] = f2_mul(a[i], w[i]);
                b[i] = f2_mul(b[i], p.interleaved ? f2_swap(wp[i]) : wp[i]);
            }
        };
        fold(p.q_weight, qa, qb);
        fold(p.k_weight, ka, kb);
    }
    const uint64_t dst0 = slot_row(p, slot) + d0, head_step = static_cast<uint64_t>(p.bs) * kHd;

#pragma unroll 1
    for (uint32_t r0 = first; r0 < rows; r0 += kRows * step) {
        load_rows(r0 + kRows * step, next);  // in flight while this pass is computed
#pragma unroll
        for (int i = 0; i < kRows; ++i) {
            const uint32_t r = r0 + i * step;
            if (r >= rows) break;
            if (r >= first_v) {
                store8(reinterpret_cast<T*>(p.v_cache) + dst0 + (r - first_v) * head_step, raw[i]);
                continue;
            }
            const bool is_k = r >= p.q_heads;
            uint64_t x[kEl / 2], y[kEl / 2];
            widen8<T>(raw[i], x);
            float scale = 1.f;
            if ((is_k ? p.k_weight : p.q_weight) != nullptr) {
                uint64_t sum2 = f2_mul(x[0], x[0]);
#pragma unroll
                for (int e = 1; e < kEl / 2; ++e) sum2 = f2_fma(x[e], x[e], sum2);
                float sum, other;
                f2_unpack(sum2, sum, other);
                sum += other;
#pragma unroll
                for (int m = LPR / 2; m > 0; m >>= 1) sum += __shfl_xor_sync(lanes, sum, m);
                scale = rsqrtf(fmaf(sum, p.inv_hd, p.eps));
            }
            if (p.interleaved) {
#pragma unroll
                for (int e = 0; e < kEl / 2; ++e) y[e] = turned != 0 ? f2_swap(x[e]) : 0;
            } else {
                Raw<T> other;
                uint32_t* to = reinterpret_cast<uint32_t*>(other.w);
                const uint32_t* from = reinterpret_cast<const uint32_t*>(raw[i].w);
#pragma unroll
                for (int e = 0; e < static_cast<int>(sizeof(Raw<T>) / 4); ++e) to[e] = __shfl_sync(lanes, from[e], partner, LPR) & turned;
                widen8<T>(other, y);
            }
            const uint64_t scale2 = f2_pack(scale, scale);
#pragma unroll
            for (int e = 0; e < kEl / 2; ++e) {
                const uint64_t b = f2_mul(y[e], is_k ? kb[e] : qb[e]);
                y[e] = f2_mul(f2_fma(x[e], is_k ? ka[e] : qa[e], b), scale2);
            }
            if (is_k) {
                store8(reinterpret_cast<T*>(p.k_cache) + dst0 + (r - p.q_heads) * head_step, narrow8<T>(y));
            } else {
                store_f8(p.q_out + (t * p.q_heads + r) * kHd + d0, y);
            }
        }
#pragma unroll
        for (int i = 0; i < kRows; ++i) raw[i] = next[i];
    }
}

// Any head size, rotary_dim and alignment: one warp per row, element by
// element; the partner element is read again (from L1). Bounded by its
// instructions, one element a lane: 8192 tokens of 32 + 8 + 8 bf16 heads of 96
// 136 us, 1.5 TB/s; 64 tokens 4.8 us.
template <typename T>
__global__ void __launch_bounds__(kAnyThreads) write_rotated_any_kernel(const __grid_constant__ RotatedParams p) {
    pdl_allow_next();
    pdl_wait();
    const int lane = threadIdx.x & 31;
    const uint64_t t = blockIdx.x;
    uint64_t pos, slot;
    if (!token_place(p, t, pos, slot)) return;
    const uint64_t dst0 = slot_row(p, slot);
    const float* tab = p.cos_sin + pos * p.rotary_dim;
    const uint32_t rot = p.rotary_dim, half = rot / 2, rows = p.q_heads + 2 * p.kv_heads;
    constexpr uint32_t kWarps = kAnyThreads / 32;
    for (uint32_t r = blockIdx.y * kWarps + threadIdx.x / 32; r < rows; r += gridDim.y * kWarps) {
        const bool is_v = r >= p.q_heads + p.kv_heads, is_k = !is_v && r >= p.q_heads;
        const uint32_t h = is_v ? r - p.q_heads - p.kv_heads : is_k ? r - p.q_heads : r;
        const T* x = is_v   ? reinterpret_cast<const T*>(p.v) + t * p.v_stride
                     : is_k ? reinterpret_cast<const T*>(p.k) + t * p.k_stride
                            : reinterpret_cast<const T*>(p.q) + t * p.q_stride;
        x += static_cast<uint64_t>(h) * p.hd;
        const uint64_t dst = dst0 + static_cast<uint64_t>(h) * p.bs * p.hd;
        if (is_v) {
            for (uint32_t d = lane; d < p.hd; d += 32) reinterpret_cast<T*>(p.v_cache)[dst + d] = x[d];
            continue;
        }
        const float* weight = is_k ? p.k_weight : p.q_weight;
        float scale = 1.f;
        if (weight != nullptr) {
            float sum = 0.f;
            for (uint32_t d = lane; d < p.hd; d += 32) {
                const float a = Elem<T>::to_f32(x[d]);
                sum = fmaf(a, a, sum);
            }
#pragma unroll
            for (int m = 16; m > 0; m >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, m);
            scale = rsqrtf(fmaf(sum, p.inv_hd, p.eps));
        }
        auto at = [&](uint32_t d) {
            const float a = Elem<T>::to_f32(x[d]);
            return weight != nullptr ? a * scale * __ldg(weight + d) : a;
        };
        for (uint32_t d = lane; d < p.hd; d += 32) {
            float y = at(d);
            if (d < rot) {
                const bool second = p.interleaved ? (d & 1u) != 0 : d >= half;
                const uint32_t i = p.interleaved ? d / 2 : (second ? d - half : d);
                const uint32_t other = p.interleaved ? d ^ 1u : (second ? d - half : d + half);
                const float c = __ldg(tab + i), s = __ldg(tab + half + i);
                y = fmaf(y, c, at(other) * (second ? s : -s));
            }
            if (is_k) {
                if constexpr (sizeof(T) == 4) reinterpret_cast<T*>(p.k_cache)[dst + d] = y;
                else reinterpret_cast<T*>(p.k_cache)[dst + d] = Elem<T>::from_f32(y);
            } else {
                p.q_out[(t * p.q_heads + h) * p.hd + d] = y;
            }
        }
    }
}

// One thread per (position, pair): the angle and its cosine and sine in FP64
// (a far position's angle loses its low bits in FP32), rounded once.
__global__ void __launch_bounds__(256) rotary_table_kernel(float* cos_sin, uint64_t total, uint32_t half,
                                                           double log2_base, double position_scale) {
    pdl_wait();
    const uint64_t stride = static_cast<uint64_t>(gridDim.x) * blockDim.x;
    for (uint64_t e = static_cast<uint64_t>(blockIdx.x) * blockDim.x + threadIdx.x; e < total; e += stride) {
        const uint64_t pos = e / half;
        const uint32_t i = static_cast<uint32_t>(e - pos * half);
        const double angle = static_cast<double>(pos) * position_scale *
                             exp2(-log2_base * static_cast<double>(i) / static_cast<double>(half));
        double s, c;
        sincos(angle, &s, &c);
        cos_sin[pos * 2 * half + i] = static_cast<float>(c);
        cos_sin[pos * 2 * half + half + i] = static_cast<float>(s);
    }
}

// A token's rows are spread over this many CTAs: one for a prefill chunk
// (which fills the GPU by its tokens), more for a decode step of few tokens.
uint32_t row_slices(uint64_t tokens, uint32_t rows, uint32_t rows_per_cta, int sms) {
    const uint64_t want = ceil_div(static_cast<uint64_t>(sms) * 4, tokens);
    return static_cast<uint32_t>(std::max<uint64_t>(1, std::min(want, ceil_div(rows, rows_per_cta))));
}

constexpr uint64_t kMaxTokens = 1ull << 30;  // per launch (grid.x)

template <typename T, int LPR>
cudaError_t launch_lpr(RotatedParams p, uint64_t n, int sms, cudaStream_t s) {
    const uint32_t rows = p.q_heads + 2 * p.kv_heads;
    const dim3 grid(static_cast<uint32_t>(n), row_slices(n, rows, kThreads / LPR, sms));
    return launch_dependent(write_rotated_kernel<T, LPR>, grid, dim3(kThreads), s, p);
}

template <typename T>
cudaError_t launch_t(const RotatedParams& p, uint64_t n, bool vec, int sms, cudaStream_t s) {
    if (vec) {
        switch (p.hd) {
        case 32: return launch_lpr<T, 4>(p, n, sms, s);
        case 64: return launch_lpr<T, 8>(p, n, sms, s);
        case 128: return launch_lpr<T, 16>(p, n, sms, s);
        case 256: return launch_lpr<T, 32>(p, n, sms, s);
        default: break;
        }
    }
    const uint32_t rows = p.q_heads + 2 * p.kv_heads;
    const dim3 grid(static_cast<uint32_t>(n), row_slices(n, rows, kAnyThreads / 32, sms));
    return launch_dependent(write_rotated_any_kernel<T>, grid, dim3(kAnyThreads), s, p);
}

bool aligned16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }
bool aligned32(const void* p) { return reinterpret_cast<uintptr_t>(p) % 32 == 0; }

}  // namespace

cudaError_t launch_write_rotated(const CacheView& c, const kvfx_rotary& rotary, const RotatedArgs& a,
                                 unsigned* status, cudaStream_t s) {
    RotatedParams p{};
    p.q_stride = a.q_stride;
    p.k_stride = a.k_stride;
    p.v_stride = a.v_stride;
    p.cos_sin = rotary.cos_sin;
    p.q_weight = rotary.q_weight;
    p.k_weight = rotary.k_weight;
    p.k_cache = c.k;
    p.v_cache = c.v;
    p.max_positions = rotary.max_positions;
    p.slot_count = c.slot_count;
    p.q_heads = a.q_heads;
    p.kv_heads = c.heads;
    p.hd = c.hd;
    p.bs = c.bs;
    p.rotary_dim = rotary.rotary_dim;
    p.interleaved = rotary.interleaved;
    p.eps = rotary.eps;
    p.inv_hd = 1.f / static_cast<float>(c.hd);
    p.status = status;
    // The vector kernel: rows of 8-element lanes, 16-byte aligned, whose
    // rotated dims end between lanes (and pair lanes with lanes).
    const uint32_t unit = 16 / c.elem;
    const bool vec = (c.hd == 32 || c.hd == 64 || c.hd == 128 || c.hd == 256) &&
                     rotary.rotary_dim % (rotary.interleaved ? kEl : 2 * kEl) == 0 && a.q_stride % unit == 0 &&
                     a.k_stride % unit == 0 && a.v_stride % unit == 0 && aligned16(a.q) && aligned16(a.k) &&
                     aligned16(a.v) && aligned32(a.q_out) && aligned16(c.k) && aligned16(c.v) &&
                     aligned16(rotary.cos_sin) && aligned16(rotary.q_weight) && aligned16(rotary.k_weight);
    const int sms = device_sm_count(c.device);
    for (uint64_t i = 0; i < a.tokens; i += kMaxTokens) {
        const uint64_t n = std::min(kMaxTokens, a.tokens - i);
        p.q = static_cast<const char*>(a.q) + i * a.q_stride * c.elem;
        p.k = static_cast<const char*>(a.k) + i * a.k_stride * c.elem;
        p.v = static_cast<const char*>(a.v) + i * a.v_stride * c.elem;
        p.positions = a.positions + i;
        p.slots = a.slots + i;
        p.q_out = a.q_out + i * a.q_heads * c.hd;
        cudaError_t e;
        switch (c.dtype) {
        case KVFX_F16: e = launch_t<__half>(p, n, vec, sms, s); break;
        case KVFX_BF16: e = launch_t<__nv_bfloat16>(p, n, vec, sms, s); break;
        default: e = launch_t<float>(p, n, vec, sms, s); break;
        }
        if (e != cudaSuccess) return e;
    }
    return cudaSuccess;
}

cudaError_t launch_rotary_table(float* cos_sin, uint64_t max_positions, uint32_t rotary_dim, double base,
                                double position_scale, cudaStream_t s) {
    const uint32_t half = rotary_dim / 2;
    const uint64_t total = max_positions * half;
    const uint32_t grid = static_cast<uint32_t>(std::min<uint64_t>(ceil_div(total, 256), 148ull * 8));
    rotary_table_kernel<<<grid, 256, 0, s>>>(cos_sin, total, half, std::log2(base), position_scale);
    return cudaGetLastError();
}

}  // namespace kvfx
