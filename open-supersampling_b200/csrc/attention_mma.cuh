// What the tensor-core attention kernels share: tile loads and stores, the bias of a tile.
#pragma once

#include <type_traits>

#include "attention.cuh"
#include "tcgen05.cuh"

namespace oss {
namespace {

constexpr int kRows = 128;  // queries of a tile

__device__ unsigned int g_timeouts;  // blocks with a wait that ran out of its limit, of this source file's kernels
__device__ __forceinline__ void count_timeout() { atomicAdd(&g_timeouts, 1u); }

__device__ __forceinline__ uint32_t pack2(float a, float b, __nv_bfloat16) {
    uint32_t r;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(b), "f"(a));
    return r;
}
__device__ __forceinline__ uint32_t pack2(float a, float b, __half) {
    uint32_t r;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(b), "f"(a));
    return r;
}

// A thread's share of the loads of one operand into panels: 16-byte chunk c of rows r0, r0 + step, ...
template <typename T, int THREADS>
struct Loader {
    const T* p;     // the head's chunk c
    int64_t st;     // token stride
    int dim, c, r0, step, shift;
    bool on, zero;  // on: the chunk belongs to the 16-column steps; zero: it lies past dim
    bool vec;       // every row starts on 16 bytes and ends on them
    bool pairs;     // on 4 bytes

    __device__ __forceinline__ Loader(const void* q, int64_t st_, int64_t sh, int dim_, int head) : st(st_), dim(dim_) {
        const int chunks = ((dim + 15) / 16) * 2;
        shift = 32 - __clz(chunks - 1);  // lanes a row: the next power of two
        c = threadIdx.x & ((1 << shift) - 1);
        r0 = (threadIdx.x & (THREADS - 1)) >> shift;
        step = THREADS >> shift;  // 8 at least, so a chunk keeps its place in the swizzle from row to row
        on = c < chunks;
        zero = c * 8 >= dim;
        p = static_cast<const T*>(q) + head * sh + (zero ? 0 : c * 8);
        vec = ((reinterpret_cast<uintptr_t>(q) & 15) | ((st_ | sh | dim) & 7)) == 0;
        pairs = ((reinterpret_cast<uintptr_t>(q) & 3) | ((st_ | sh | dim) & 1)) == 0;
    }
    __device__ __forceinline__ uint32_t place(uint32_t dst, int panel_rows) const {
        return dst + (c >> 3) * panel_rows * 128 + r0 * 128 + (((c & 7) ^ (r0 & 7)) << 4);
    }
    // `rows` rows from token on, zeros from there to rows_pad; of the head `skip` elements further.
    __device__ __forceinline__ void load(uint32_t dst, int panel_rows, int64_t token, int rows, int rows_pad, int64_t skip = 0) const {
        if (!on) return;
        uint32_t to = place(dst, panel_rows);
        const T* from = p + (token + r0) * st + skip;
        int r = r0;
        if (!zero) {
            if (vec) {
                for (; r < rows; r += step, to += step * 128, from += step * st) tc::cp_async16(to, from);
            } else {
                for (; r < rows; r += step, to += step * 128, from += step * st) store_some(to, from);
            }
        }
        for (; r < rows_pad; r += step, to += step * 128) store_zero(to);
    }
    // The same for rows that are the heads of a group: row r is token r / pack, head r % pack.
    __device__ __forceinline__ void load_packed(uint32_t dst, int panel_rows, int64_t token, int64_t sh, int pack, int first, int rows,
                                                int rows_pad) const {
        if (!on) return;
        uint32_t to = place(dst, panel_rows);
        for (int r = r0; r < rows_pad; r += step, to += step * 128) {
            const T* from = p + (token + (first + r) / pack) * st + (first + r) % pack * sh;
            if (zero || r >= rows)
                store_zero(to);
            else if (vec)
                tc::cp_async16(to, from);
            else
                store_some(to, from);
        }
    }
    __device__ __forceinline__ static void store_zero(uint32_t to) {
        asm volatile("st.shared.v4.b32 [%0], {%1,%1,%1,%1};" ::"r"(to), "r"(0) : "memory");
    }
    __device__ __forceinline__ void store_some(uint32_t to, const T* from) const {
        if (pairs) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                if (c * 8 + 2 * e < dim)
                    tc::cp_async4(to + 4 * e, from + 2 * e);
                else
                    asm volatile("st.shared.b32 [%0], %1;" ::"r"(to + 4 * e), "r"(0) : "memory");
            }
            return;
        }
        uint32_t w[4] = {0, 0, 0, 0};
        const unsigned short* s = reinterpret_cast<const unsigned short*>(from);
#pragma unroll
        for (int e = 0; e < 8; ++e)
            if (c * 8 + e < dim) w[e >> 1] |= static_cast<uint32_t>(__ldg(s + e)) << (16 * (e & 1));
        asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};" ::"r"(to), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]) : "memory");
    }
};

// ---- bias of a tile ----------------------------------------------------------------
// How the entries of a tile of queries x keys are found. Most tiles need no clamping: windows
// never leave the map, and far tokens all clamp to one entry.
enum BiasMode { kLinear, kLinearX, kClamp, kOne };

struct Range {  // of positions
    int y0, y1, x0, x1;
};
__device__ __forceinline__ BiasMode bias_mode(const AttnBias& b, const Range& q, const Range& k) {
    const int ylo = k.y0 - q.y1, yhi = k.y1 - q.y0, xlo = k.x0 - q.x1, xhi = k.x1 - q.x0;
    const bool yin = ylo >= -b.ry && yhi <= b.ry, xin = xlo >= -b.rx && xhi <= b.rx;
    const bool yone = ylo >= b.ry || yhi <= -b.ry, xone = xlo >= b.rx || xhi <= -b.rx;
    if (yone && xone) return kOne;
    if (yone && xin) return kLinearX;
    return yin && xin ? kLinear : kClamp;
}
__device__ __forceinline__ Range warp_range(int2 p) {
    return {__reduce_min_sync(0xffffffffu, p.x), __reduce_max_sync(0xffffffffu, p.x), __reduce_min_sync(0xffffffffu, p.y),
            __reduce_max_sync(0xffffffffu, p.y)};
}
__device__ __forceinline__ Range join(const Range& a, const Range& b) {
    return {min(a.y0, b.y0), max(a.y1, b.y1), min(a.x0, b.x0), max(a.x1, b.x1)};
}

// y (2 rx + 1) + x; wraps where nobody uses it.
__device__ __forceinline__ int linear_code(const AttnBias& b, int y, int x) {
    return static_cast<int>(static_cast<unsigned>(y) * static_cast<unsigned>(2 * b.rx + 1) + static_cast<unsigned>(x));
}

template <int KT>
struct KeyPos {  // of a tile, in shared memory
    int y[KT], x[KT], code[KT];  // code: (y - y[0]) (2 rx + 1) + x, of use where no pair needs clamping
    Range range[KT / 32];
};

// Fills it; threads 0 .. KT - 1. n > 0 live keys.
template <int KT>
__device__ __forceinline__ void load_key_pos(KeyPos<KT>* s, const AttnBias& b, int64_t token, int n) {
    const int j = threadIdx.x;
    if (j >= KT) return;
    const int2 p = bias_pos(b.k_pos, b.axes, token + min(j, n - 1));
    s->y[j] = p.x;
    s->x[j] = p.y;
    s->code[j] = linear_code(b, p.x - bias_pos(b.k_pos, b.axes, token).x, p.y);
    const Range r = warp_range(p);
    if ((j & 31) == 0) s->range[j >> 5] = r;
}
// The same by one warp.
template <int KT>
__device__ __forceinline__ void load_key_pos_warp(KeyPos<KT>* s, const AttnBias& b, int64_t token, int n) {
#pragma unroll
    for (int w = 0; w < KT / 32; ++w) {
        const int j = 32 * w + (threadIdx.x & 31), y0 = bias_pos(b.k_pos, b.axes, token).x;
        const int2 p = bias_pos(b.k_pos, b.axes, token + min(j, n - 1));
        s->y[j] = p.x;
        s->x[j] = p.y;
        s->code[j] = linear_code(b, p.x - y0, p.y);
        const Range r = warp_range(p);
        if ((j & 31) == 0) s->range[w] = r;
    }
}
template <int KT>
__device__ __forceinline__ Range key_range(const KeyPos<KT>* s) {
    Range r = s->range[0];
#pragma unroll
    for (int w = 1; w < KT / 32; ++w) r = join(r, s->range[w]);
    return r;
}

// x[c] = x[c] c2 + bias of keys j0 + c, for a row at qp; keys up to n16 of the tile.
template <int KT, int N>
__device__ __forceinline__ void add_bias(float (&x)[N], float c2, const AttnBias& b, BiasMode mode, const float* E,
                                         const KeyPos<KT>* k, int j0, int n16, int2 qp) {
    const int w = 2 * b.rx + 1;
    if (mode == kOne) {
        const float e = E[bias_index(b, qp, make_int2(k->y[0], k->x[0]))];
        const float2 by = make_float2(c2, c2), add = make_float2(e, e);
#pragma unroll
        for (int c = 0; c < N; c += 2) {
            const float2 y = __ffma2_rn(make_float2(x[c], x[c + 1]), by, add);
            x[c] = y.x;
            x[c + 1] = y.y;
        }
    } else if (mode == kClamp) {
#pragma unroll
        for (int c = 0; c < N; ++c)
            if (j0 + (c & ~15) < n16) x[c] = fmaf(x[c], c2, E[bias_index(b, qp, make_int2(k->y[j0 + c], k->x[j0 + c]))]);
    } else {
        const int* code = mode == kLinear ? k->code + j0 : k->x + j0;
        const int dy = min(max(k->y[0] - qp.x, -b.ry), b.ry);
        const float* at = E + (dy + b.ry) * w + b.rx - qp.y;
#pragma unroll
        for (int c = 0; c < N; c += 4) {
            if (j0 + (c & ~15) >= n16) continue;
            const int4 q = *reinterpret_cast<const int4*>(code + c);
            x[c] = fmaf(x[c], c2, at[q.x]);
            x[c + 1] = fmaf(x[c + 1], c2, at[q.y]);
            x[c + 2] = fmaf(x[c + 2], c2, at[q.z]);
            x[c + 3] = fmaf(x[c + 3], c2, at[q.w]);
        }
    }
}

// 16 columns of a row of an output tile, times `by`, into the panels at dst.
template <typename T>
__device__ __forceinline__ void stage16(uint32_t dst, int r, const float* o, int c, float by) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = pack2(o[8 * h + 2 * i] * by, o[8 * h + 2 * i + 1] * by, T{});
        const int chunk = (c >> 3) + h;
        const uint32_t to = dst + (chunk >> 3) * kRows * 128 + r * 128 + (((chunk & 7) ^ (r & 7)) << 4);
        asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};" ::"r"(to), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]) : "memory");
    }
}
// Rows of a staged tile to memory, whole rows together; row r is token (first + r) / pack.
template <typename T, int THREADS>
__device__ __forceinline__ void store_panel(uint32_t src0, void* out, int heads, int dim, int64_t token0, int head0, int pack,
                                            int first, int rows) {
    const int chunks = (dim + 7) / 8, shift = chunks > 1 ? 32 - __clz(chunks - 1) : 0;
    const int c = threadIdx.x & ((1 << shift) - 1), step = THREADS >> shift;
    if (c >= chunks) return;
    const bool vec = (reinterpret_cast<uintptr_t>(out) & 15) == 0 && dim % 8 == 0;
    const bool pairs = (reinterpret_cast<uintptr_t>(out) & 3) == 0 && dim % 2 == 0;
    for (int r = threadIdx.x >> shift; r < rows; r += step) {
        const int64_t row = pack == 1 ? (token0 + first + r) * heads + head0
                                      : (token0 + (first + r) / pack) * heads + head0 + (first + r) % pack;
        const uint32_t src = src0 + (c >> 3) * kRows * 128 + r * 128 + (((c & 7) ^ (r & 7)) << 4);
        uint32_t w[4];
        asm volatile("ld.shared.v4.b32 {%0,%1,%2,%3}, [%4];" : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "r"(src));
        unsigned short* dst = static_cast<unsigned short*>(out) + row * dim + c * 8;
        if (vec) {
            *reinterpret_cast<uint4*>(dst) = make_uint4(w[0], w[1], w[2], w[3]);
        } else if (pairs) {
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (c * 8 + 2 * e < dim) reinterpret_cast<uint32_t*>(dst)[e] = w[e];
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e)
                if (c * 8 + e < dim) dst[e] = static_cast<unsigned short>(w[e >> 1] >> (16 * (e & 1)));
        }
    }
}
__device__ __forceinline__ void write_part(float* to, const float* o, int c, int dim) {
    if ((dim & 3) == 0) {
#pragma unroll
        for (int i = 0; i < 16; i += 4)
            if (c + i < dim) *reinterpret_cast<float4*>(to + c + i) = make_float4(o[i], o[i + 1], o[i + 2], o[i + 3]);
    } else {
#pragma unroll
        for (int i = 0; i < 16; ++i)
            if (c + i < dim) to[c + i] = o[i];
    }
}

// ---- what a mask hides --------------------------------------------------------------
// A hidden weight of 0 times a NaN or an infinity is NaN. Rows that come out not finite are found again from
// what they see, one thread a row; but only where that can help: where something hidden is not finite, and
// nothing that is seen explains it. In a causal window these are rows within a tile of the first such value,
// however many values are not finite. 4096 tokens, 2 heads of 64, forward and backward: 0.4 ms with a NaN in the
// first key, as without (82 ms with every row found again), 3.6 ms with an infinity in the middle value.

// The last of rows [from, to) with a value that is not finite, or -1. A whole warp.
template <typename T>
__device__ __noinline__ int last_not_finite(const T* x, int64_t st, int from, int to, int dim) {
    int last = -1;
    for (int c = threadIdx.x & 31; c < dim; c += 32)
#pragma unroll 8
        for (int r = from; r < to; ++r)
            if (!is_finite(to_f(x[r * st + c]))) last = max(last, r);
    return __reduce_max_sync(0xffffffffu, last);
}
// Some column has a value that is not finite among the hidden rows [h0, h1), and none among the seen rows [s0, s1).
template <typename T>
__device__ __noinline__ bool hidden_spoils(const T* x, int64_t st, int h0, int h1, int s0, int s1, int dim) {
    for (int c = 0; c < dim; ++c) {
        bool hidden = false, seen = false;
        for (int r = h0; r < h1 && !hidden; ++r) hidden = !is_finite(to_f(x[r * st + c]));
        if (!hidden) continue;
        for (int r = s1 - 1; r >= s0 && !seen; --r) seen = !is_finite(to_f(x[r * st + c]));
        if (!seen) return true;
    }
    return false;
}

template <typename T>
constexpr int kIsBf16 = std::is_same<T, __nv_bfloat16>::value ? 1 : 0;

// Power of two that dS of a window and key head is kept times. (One for the whole call let a large value
// in another window, or in a row that no window holds, push dS below fp16's range.)
template <typename T>
__device__ __forceinline__ float ds_scale(const AttnParams& p, int window, int kvh) {
    if constexpr (kIsBf16<T>) return 1.0f;
    const uint2 m = __ldg(reinterpret_cast<const uint2*>(p.win_max) + static_cast<int64_t>(window) * p.kv_heads + kvh);
    const float most_do = __half2float(__ushort_as_half(static_cast<unsigned short>(m.x))),
                most_v = __half2float(__ushort_as_half(static_cast<unsigned short>(m.y)));
    const float bound = 2.0f * p.dim * most_do * most_v;
    if (!(bound > 0.0f)) return 1.0f;
    return exp2f(static_cast<float>(min(max(14 - ilogbf(bound), -100), 100)));
}

}  // namespace
}  // namespace oss
