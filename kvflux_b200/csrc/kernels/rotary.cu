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
// with the token's cosines and sines in registers; all of a pass's rows are
// loaded before the first is used. The norm's sum and the rotation's partner
// dims move by shuffles inside the group.
#include <algorithm>
#include <cmath>

#include "common.cuh"
#include "launch.h"

namespace kvfx {
namespace {

constexpr int kThreads = 128;
constexpr int kEl = 8;    // elements per lane
constexpr int kRows = 4;  // rows in flight per lane group

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
    uint64_t tokens, max_positions, slot_count;
    uint32_t q_heads, kv_heads, hd, bs, rotary_dim, interleaved;
    float eps, inv_hd;
    unsigned* status;
};

template <typename T>
__device__ __forceinline__ void load8(const T* p, uint4 (&raw)[sizeof(T) / 2]) {
#pragma unroll
    for (int i = 0; i < static_cast<int>(sizeof(T) / 2); ++i) raw[i] = __ldg(reinterpret_cast<const uint4*>(p) + i);
}

template <typename T>
__device__ __forceinline__ void widen8(const uint4 (&raw)[sizeof(T) / 2], float (&x)[kEl]) {
    const T* e = reinterpret_cast<const T*>(raw);
#pragma unroll
    for (int i = 0; i < kEl; ++i) x[i] = Elem<T>::to_f32(e[i]);
}

template <typename T>
__device__ __forceinline__ void narrow8(const float (&x)[kEl], uint4 (&raw)[sizeof(T) / 2]) {
    if constexpr (sizeof(T) == 2) {
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = Elem<T>::pack(x[2 * i], x[2 * i + 1]);
        raw[0] = make_uint4(w[0], w[1], w[2], w[3]);
    } else {
#pragma unroll
        for (int i = 0; i < 2; ++i)
            raw[i] = make_uint4(__float_as_uint(x[4 * i]), __float_as_uint(x[4 * i + 1]),
                                __float_as_uint(x[4 * i + 2]), __float_as_uint(x[4 * i + 3]));
    }
}

template <typename T>
__device__ __forceinline__ void store8(T* p, const uint4 (&raw)[sizeof(T) / 2]) {
#pragma unroll
    for (int i = 0; i < static_cast<int>(sizeof(T) / 2); ++i) reinterpret_cast<uint4*>(p)[i] = raw[i];
}

__device__ __forceinline__ void load_f8(const float* p, float (&x)[kEl]) {
#pragma unroll
    for (int i = 0; i < kEl / 4; ++i) {
        const float4 a = __ldg(reinterpret_cast<const float4*>(p) + i);
        x[4 * i] = a.x;
        x[4 * i + 1] = a.y;
        x[4 * i + 2] = a.z;
        x[4 * i + 3] = a.w;
    }
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

// LPR lanes per row (head_size = 8 LPR). One CTA per token and slice of its
// rows (blockIdx.y of gridDim.y); rows are Q heads, K heads, V heads in turn.
template <typename T, int LPR>
__global__ void __launch_bounds__(kThreads) write_rotated_kernel(const __grid_constant__ RotatedParams p) {
    constexpr int kGroups = kThreads / LPR;
    constexpr int kHd = LPR * kEl;
    pdl_allow_next();
    pdl_wait();  // launched as a dependent: the previous kernel's writes first
    const uint64_t t = blockIdx.x;
    const int l = threadIdx.x % LPR, g = threadIdx.x / LPR;
    const uint32_t rows = p.q_heads + 2 * p.kv_heads;
    const uint32_t first = blockIdx.y * kGroups + g, step = gridDim.y * kGroups;
    const int d0 = l * kEl;

    auto row_ptr = [&](uint32_t r) {
        const T* base = reinterpret_cast<const T*>(p.q) + t * p.q_stride;
        uint32_t h = r;
        if (r >= p.q_heads + p.kv_heads) {
            base = reinterpret_cast<const T*>(p.v) + t * p.v_stride;
            h = r - p.q_heads - p.kv_heads;
        } else if (r >= p.q_heads) {
            base = reinterpret_cast<const T*>(p.k) + t * p.k_stride;
            h = r - p.q_heads;
        }
        return base + static_cast<uint64_t>(h) * kHd + d0;
    };
    uint4 raw[kRows][sizeof(T) / 2];
    auto load_rows = [&](uint32_t r0) {
#pragma unroll
        for (int i = 0; i < kRows; ++i) {
            const uint32_t r = r0 + i * step;
            if (r < rows) load8(row_ptr(r), raw[i]);
        }
    };
    load_rows(first);  // independent of the token's place: both latencies overlap
    uint64_t pos, slot;
    if (!token_place(p, t, pos, slot)) return;

    // This lane's rotation: y = x * c + partner * s.
    const int rot = static_cast<int>(p.rotary_dim), half = rot / 2;
    float c[kEl], s[kEl];
    int partner = l;
    const float* tab = p.cos_sin + pos * p.rotary_dim;
#pragma unroll
    for (int i = 0; i < kEl; ++i) {
        c[i] = 1.f;
        s[i] = 0.f;
    }
    if (p.interleaved) {  // pairs (2i, 2i + 1): four angles, partner in the same lane
        if (d0 < rot) {
            const float4 cc = __ldg(reinterpret_cast<const float4*>(tab + d0 / 2));
            const float4 ss = __ldg(reinterpret_cast<const float4*>(tab + half + d0 / 2));
            c[0] = c[1] = cc.x, c[2] = c[3] = cc.y, c[4] = c[5] = cc.z, c[6] = c[7] = cc.w;
            s[0] = -ss.x, s[1] = ss.x, s[2] = -ss.y, s[3] = ss.y;
            s[4] = -ss.z, s[5] = ss.z, s[6] = -ss.w, s[7] = ss.w;
        }
    } else if (d0 < rot) {  // pairs (i, i + rot / 2): the partner lane holds the other half
        const bool low = d0 < half;
        partner = low ? l + half / kEl : l - half / kEl;
        const int a0 = low ? d0 : d0 - half;
        load_f8(tab + a0, c);
        load_f8(tab + half + a0, s);
        if (low) {
#pragma unroll
            for (int i = 0; i < kEl; ++i) s[i] = -s[i];
        }
    }
    float wq[kEl], wk[kEl];
    if (p.q_weight != nullptr) load_f8(p.q_weight + d0, wq);
    if (p.k_weight != nullptr) load_f8(p.k_weight + d0, wk);

    const uint64_t page = slot / p.bs, off = slot - page * p.bs;
    // Rows in passes of kRows per group; every lane takes the same number of
    // passes (shuffles below), rows past the end are not stored.
    for (uint32_t r0 = first; r0 - g < rows; r0 += kRows * step) {
        if (r0 != first) load_rows(r0);
#pragma unroll
        for (int i = 0; i < kRows; ++i) {
            const uint32_t r = r0 + i * step;
            const bool is_v = r >= p.q_heads + p.kv_heads, is_k = !is_v && r >= p.q_heads;
            if (r - g >= rows) break;  // past the end for every lane of the CTA
            float x[kEl], y[kEl];
            widen8<T>(raw[i], x);
            const float* weight = is_k ? p.k_weight : p.q_weight;
            float sum = 0.f;
#pragma unroll
            for (int e = 0; e < kEl; ++e) sum = fmaf(x[e], x[e], sum);
#pragma unroll
            for (int m = LPR / 2; m > 0; m >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, m);
            if (weight != nullptr) {
                const float scale = rsqrtf(fmaf(sum, p.inv_hd, p.eps));
#pragma unroll
                for (int e = 0; e < kEl; ++e) x[e] = x[e] * scale * (is_k ? wk[e] : wq[e]);
            }
            if (p.interleaved) {
#pragma unroll
                for (int e = 0; e < kEl; ++e) y[e] = fmaf(x[e], c[e], x[e ^ 1] * s[e]);
            } else {
#pragma unroll
                for (int e = 0; e < kEl; ++e) {
                    const float other = __shfl_sync(0xffffffffu, x[e], partner, LPR);
                    y[e] = fmaf(x[e], c[e], other * s[e]);
                }
            }
            if (r >= rows) continue;
            if (r < p.q_heads) {
                float4* out = reinterpret_cast<float4*>(p.q_out + (t * p.q_heads + r) * kHd + d0);
                out[0] = make_float4(y[0], y[1], y[2], y[3]);
                out[1] = make_float4(y[4], y[5], y[6], y[7]);
                continue;
            }
            const uint32_t h = r - p.q_heads - (is_v ? p.kv_heads : 0);
            const uint64_t dst = ((page * p.kv_heads + h) * p.bs + off) * kHd + d0;
            if (is_v) {
                store8(reinterpret_cast<T*>(p.v_cache) + dst, raw[i]);
            } else {
                uint4 k8[sizeof(T) / 2];
                narrow8<T>(y, k8);
                store8(reinterpret_cast<T*>(p.k_cache) + dst, k8);
            }
        }
    }
}

// Any head size, rotary_dim and alignment: one warp per row, element by
// element; the partner element is read again (from L1).
template <typename T>
__global__ void __launch_bounds__(kThreads) write_rotated_any_kernel(const __grid_constant__ RotatedParams p) {
    pdl_allow_next();
    pdl_wait();
    const int lane = threadIdx.x & 31;
    const uint64_t t = blockIdx.x;
    uint64_t pos, slot;
    if (!token_place(p, t, pos, slot)) return;
    const uint64_t page = slot / p.bs, off = slot - page * p.bs;
    const float* tab = p.cos_sin + pos * p.rotary_dim;
    const uint32_t rot = p.rotary_dim, half = rot / 2, rows = p.q_heads + 2 * p.kv_heads;
    constexpr uint32_t kWarps = kThreads / 32;
    for (uint32_t r = blockIdx.y * kWarps + threadIdx.x / 32; r < rows; r += gridDim.y * kWarps) {
        const bool is_v = r >= p.q_heads + p.kv_heads, is_k = !is_v && r >= p.q_heads;
        const uint32_t h = is_v ? r - p.q_heads - p.kv_heads : is_k ? r - p.q_heads : r;
        const T* x = is_v   ? reinterpret_cast<const T*>(p.v) + t * p.v_stride
                     : is_k ? reinterpret_cast<const T*>(p.k) + t * p.k_stride
                            : reinterpret_cast<const T*>(p.q) + t * p.q_stride;
        x += static_cast<uint64_t>(h) * p.hd;
        const uint64_t dst = ((page * p.kv_heads + h) * p.bs + off) * p.hd;
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
    const dim3 grid(static_cast<uint32_t>(n), row_slices(n, rows, kThreads / 32, sms));
    return launch_dependent(write_rotated_any_kernel<T>, grid, dim3(kThreads), s, p);
}

bool aligned16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

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
                     aligned16(a.v) && aligned16(a.q_out) && aligned16(c.k) && aligned16(c.v) &&
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
        p.tokens = n;
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
