// Window attention of 16-bit types on the tensor cores (tcgen05): backward.
//
// Per tile of 128 queries x keys, with 32 keys of a query row for each thread:
//   S = Q K^T, dP = dO V^T          into tensor memory
//   P = 2^(S - lse), dS = P (dP - delta)   in registers, written to shared memory as 16-bit values
//   dV += P^T dO, dK += dS^T Q, dQ += dS K from shared memory: a row-major P is a K-major operand for
//                                   dQ and an MN-major one for the other two, so nothing is transposed
//
// Windows of up to 64 keys (the Gaussians of a tile) take one kernel: a block holds the window's
// keys and walks its queries, so that q, k, v and dout are read once and every gradient leaves
// the block finished; delta comes from the row of P and dP itself. Longer windows take two, one
// that walks keys for dQ and one that walks queries for dK and dV (seven products instead of five,
// but no sums across blocks: every gradient has a fixed order of additions).
//
// fp16 keeps dS times a power of two that puts the window's bound 2 dim max|dout| max|v| at 2^15, so that
// gradients of any size stay within the type's range.
//
// The bias gradient is summed per tile in shared 32-bit integers (native atomics; the same in any
// order) at 2^-30 of the tile's sum of |dS|, which no entry exceeds, and then in fp64 by the entry's
// own thread. Blocks keep their head and their tiles from run to run; their sums are added in order
// at the end.
#include "attention_mma.cuh"
#include "internal.h"

namespace oss {
namespace {

constexpr int kShortKeys = 64;

constexpr float kNaN = __builtin_nanf("");

// The end of a block. Where a wait has run out (`lost`): counted, and what is still in flight is waited for.
__device__ __forceinline__ void finish_block(bool lost, uint32_t bar_end) {
    if (lost) {
        tc::cp_async_wait<0>();
        if (threadIdx.x == 0) count_timeout();
        if (threadIdx.x < 32) {
            if (tc::elect_one()) tc::commit(bar_end);
            __syncwarp();
            tc::mbar_settle(bar_end, 0);
        }
    }
    __syncthreads();
}

struct BiasSum {      // of a tile, uniform over the block
    BiasMode mode;
    float fixed;      // 0: nothing to add
    bool bad;         // some terms are not finite
};

template <int WARPS>
__device__ __forceinline__ BiasSum bias_sum(BiasMode mode, const float* wsize) {
    float m = 0.0f;
    bool bad = false;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) {
        m += fabsf(wsize[w]);
        bad |= wsize[w] < 0.0f;
    }
    BiasSum b{mode, 0.0f, bad};
    b.fixed = bias_scale(m, 30);
    return b;
}

// Adds a thread's terms of keys j0 .. to the block's integers (wsum: a warp's sum where the tile
// has one entry).
template <int KT, int N>
__device__ __forceinline__ void bias_add(const AttnParams& p, const BiasSum& b, const float (&ds)[N], int n16, int head,
                                         const KeyPos<KT>* k, int j0, int2 qp, int* I, float* wsum) {
    if (b.mode == kOne) {
        float sum = 0.0f;
#pragma unroll
        for (int c = 0; c < N; ++c) sum += ds[c];  // 0 past the last key
#pragma unroll
        for (int x = 16; x > 0; x >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, x);
        if ((threadIdx.x & 31) == 0) *wsum = sum;
        return;
    }
    if (b.bad || b.mode == kClamp) {
#pragma unroll
        for (int c = 0; c < N; ++c) {
            if (j0 + c >= n16) break;
            const int e = bias_index(p.bias, qp, make_int2(k->y[j0 + c], k->x[j0 + c]));
            if (!is_finite(ds[c]))
                bias_mark_bad(p, head, e);
            else
                atomicAdd(I + e, __float2int_rn(ds[c] * b.fixed));
        }
        return;
    }
    const int w = 2 * p.bias.rx + 1;
    const int* code = b.mode == kLinear ? k->code + j0 : k->x + j0;
    const int dy = min(max(k->y[0] - qp.x, -p.bias.ry), p.bias.ry);
    int* at = I + (dy + p.bias.ry) * w + p.bias.rx - qp.y;
#pragma unroll
    for (int c = 0; c < N; c += 4) {
        if (j0 + c >= n16) break;
        const int4 q = *reinterpret_cast<const int4*>(code + c);
        atomicAdd(at + q.x, __float2int_rn(ds[c] * b.fixed));
        atomicAdd(at + q.y, __float2int_rn(ds[c + 1] * b.fixed));
        atomicAdd(at + q.z, __float2int_rn(ds[c + 2] * b.fixed));
        atomicAdd(at + q.w, __float2int_rn(ds[c + 3] * b.fixed));
    }
}

// After a barrier: the integers join the block's fp64 sums.
template <int THREADS, int WARPS, int KT>
__device__ __forceinline__ void bias_join(const AttnParams& p, const BiasSum& b, int entries, int head, const KeyPos<KT>* k,
                                          int2 qp, int* I, const float* wsum, double* acc) {
    if (b.mode == kOne) {
        if (threadIdx.x == 0) {
            const int e = bias_index(p.bias, qp, make_int2(k->y[0], k->x[0]));
            double sum = 0.0;
#pragma unroll
            for (int w = 0; w < WARPS; ++w) sum += static_cast<double>(wsum[w]);
            if (b.bad)
                bias_mark_bad(p, head, e);
            else
                acc[e] += sum;
        }
        return;
    }
    if (b.fixed == 0.0f) return;
    const double unit = 1.0 / static_cast<double>(b.fixed);
    for (int e = threadIdx.x; e < entries; e += THREADS) {
        const int v = I[e];
        if (v != 0) {
            acc[e] += static_cast<double>(v) * unit;
            I[e] = 0;
        }
    }
}

// N values of a row, columns j0 .., as 16-bit into panels.
template <typename T, int N>
__device__ __forceinline__ void write_row(uint32_t panels, int row, int j0, const float (&x)[N], float by) {
    const uint32_t panel = panels + (j0 >> 6) * kRows * 128, chunk0 = (j0 & 63) >> 3;
#pragma unroll
    for (int c = 0; c < N; c += 8) {
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = pack2(x[c + 2 * i] * by, x[c + 2 * i + 1] * by, T{});
        const uint32_t to = panel + row * 128 + (((chunk0 + (c >> 3)) ^ (row & 7)) << 4);
        asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};" ::"r"(to), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]) : "memory");
    }
}

// 16 columns of a row of a gradient, straight to memory.
template <typename T>
__device__ __forceinline__ void write_out(T* to, const float* o, int c, int dim, float by) {
    if (dim % 8 == 0 && (reinterpret_cast<uintptr_t>(to) & 15) == 0) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            if (c + 8 * h >= dim) continue;
            uint32_t w[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) w[i] = pack2(o[8 * h + 2 * i] * by, o[8 * h + 2 * i + 1] * by, T{});
            *reinterpret_cast<uint4*>(to + c + 8 * h) = make_uint4(w[0], w[1], w[2], w[3]);
        }
    } else if (dim % 2 == 0 && (reinterpret_cast<uintptr_t>(to) & 3) == 0) {
#pragma unroll
        for (int i = 0; i < 16; i += 2)
            if (c + i < dim) reinterpret_cast<uint32_t*>(to + c)[i / 2] = pack2(o[i] * by, o[i + 1] * by, T{});
    } else {
#pragma unroll
        for (int i = 0; i < 16; ++i)
            if (c + i < dim) to[c + i] = from_f<T>(o[i] * by);
    }
}

// Scores and dP of a thread's N keys from tensor memory, and the weights: s becomes p, dp stays.
// Zero where the mask is, whatever stands there.
template <int KT, bool BIAS, int N>
__device__ __forceinline__ void weights(const AttnParams& p, float (&s)[N], float (&dp)[N], uint32_t ts, uint32_t tdp, int n16,
                                        int j0, bool whole, int see, float lse, float far, BiasMode mode, const float* E,
                                        const KeyPos<KT>* kp, int2 qp) {
    const float c2 = p.scale * kLog2e;
#pragma unroll
    for (int c = 0; c < N; c += 16) {
        if (j0 + c < n16) {
            tc::tmem_ld16(ts + j0 + c, s + c);
            tc::tmem_ld16(tdp + j0 + c, dp + c);
        } else {
#pragma unroll
            for (int i = 0; i < 16; ++i) s[c + i] = dp[c + i] = 0.0f;
        }
    }
    tc::wait_ld();
    const float2 by = make_float2(BIAS ? 1.0f : c2, BIAS ? 1.0f : c2), off = make_float2(-lse, -lse);
    if constexpr (BIAS) add_bias<KT>(s, c2, p.bias, mode, E, kp, j0, n16, qp);
#pragma unroll
    for (int c = 0; c < N; c += 16) {
        if (j0 + c >= n16) {  // nothing of the bias stays there
#pragma unroll
            for (int i = 0; i < 16; ++i) s[c + i] = 0.0f;
            continue;
        }
#pragma unroll
        for (int i = 0; i < 16; i += 2) {
            const float2 x = make_float2(s[c + i], s[c + i + 1]), y = BIAS ? __fadd2_rn(x, off) : __ffma2_rn(x, by, off);
            s[c + i] = ex2(y.x);
            s[c + i + 1] = ex2(y.y);
        }
    }
    if (__any_sync(0xffffffffu, far != 1.0f)) {
#pragma unroll
        for (int c = 0; c < N; ++c) s[c] *= far;
    }
    if (!whole) {
#pragma unroll
        for (int c = 0; c < N; ++c) {
            const bool on = j0 + c < see;
            s[c] = on ? s[c] : 0.0f;
            dp[c] = on ? dp[c] : 0.0f;
        }
    }
}

// dp becomes p (dp - delta). Hidden pairs' are 0 even where delta is not finite.
template <int N>
__device__ __forceinline__ void score_gradients(const float (&s)[N], float (&dp)[N], float delta, int j0, bool whole, int see) {
    const float2 off = make_float2(-delta, -delta);
#pragma unroll
    for (int c = 0; c < N; c += 2) {
        const float2 d = __fmul2_rn(make_float2(s[c], s[c + 1]), __fadd2_rn(make_float2(dp[c], dp[c + 1]), off));
        dp[c] = d.x;
        dp[c + 1] = d.y;
    }
    if (!whole) {
#pragma unroll
        for (int c = 0; c < N; ++c) dp[c] = j0 + c < see ? dp[c] : 0.0f;
    }
}

// ---- rows again, where a product met what its mask hides ------------------------------------
template <typename T>
__device__ __forceinline__ float dot_row(const T* a, const T* b, int dim) {
    float s = 0.0f;
    for (int c = 0; c < dim; ++c) s = fmaf(to_f(a[c]), to_f(b[c]), s);
    return s;
}
template <typename T>
__device__ __forceinline__ float score_of(const AttnParams& p, int64_t q, int64_t k, int head, int kvh) {
    float s = dot_row(static_cast<const T*>(p.q) + q * p.q_st + head * p.q_sh, static_cast<const T*>(p.k) + k * p.k_st + kvh * p.k_sh,
                      p.dim) * (p.scale * kLog2e);
    if (p.bias.table != nullptr)
        s += bias_entry(p.bias, p.heads, head, bias_index(p.bias, bias_pos(p.bias.q_pos, p.bias.axes, q), bias_pos(p.bias.k_pos, p.bias.axes, k)));
    return s;
}

// dq of one row over the keys [k0, k0 + see) that it sees, staged in the panels at `stage`.
template <typename T>
__device__ __noinline__ void query_row(const AttnParams& p, int64_t q, int head, int64_t k0, int see, float lse, float far, float delta, float up,
                                       uint32_t stage) {
    float o[kMaxHeadDim];
    const int kvh = head / (p.heads / p.kv_heads);
    const T* g = static_cast<const T*>(p.dout) + q * p.do_st + head * p.do_sh;
    for (int c = 0; c < kMaxHeadDim; ++c) o[c] = 0.0f;
    for (int64_t k = k0; k < k0 + see; ++k) {
        const float w = ex2(score_of<T>(p, q, k, head, kvh) - lse) * far;
        const float d = to_f(from_f<T>(w * (dot_row(g, static_cast<const T*>(p.v) + k * p.v_st + kvh * p.v_sh, p.dim) - delta) * up));
        const T* kk = static_cast<const T*>(p.k) + k * p.k_st + kvh * p.k_sh;
        for (int c = 0; c < p.dim; ++c) o[c] = fmaf(d, to_f(kk[c]), o[c]);
    }
    for (int c = 0; c < ((p.dim + 15) & ~15); c += 16) stage16<T>(stage, threadIdx.x & (kRows - 1), o + c, c, p.scale / up);
}

// Whether query_row has to find dq again: dq came out not finite (`odd`) with finite weights. Whole warps; row of the lane.
template <typename T>
__device__ __forceinline__ bool query_again(const AttnParams& p, bool odd, int64_t k0, int kvh, int see, int most, float lse, float delta) {
    bool again = odd && (see == 0 || (is_finite(lse) && is_finite(delta)));
    if (__any_sync(0xffffffffu, again)) {
        const T* kb = static_cast<const T*>(p.k) + k0 * p.k_st + kvh * p.k_sh;
        const int last = last_not_finite<T>(kb, p.k_st, __reduce_min_sync(0xffffffffu, again ? see : most), most, p.dim);
        again = again && last >= see && hidden_spoils<T>(kb, p.k_st, see, last + 1, 0, see, p.dim);
    }
    return again;
}

// Whether key_row has to find dk (want_v: dv) of the j-th key again, whose products began with query tile qt0 of a
// head. Whole warps; key of the lane.
template <typename T>
__device__ __noinline__ bool key_again(const AttnParams& p, bool odd, int j, int kvh, int64_t q0, int lq, int lk, int qt0, int i0, int i1,
                                       bool want_v) {
    if (!__any_sync(0xffffffffu, odd)) return false;
    const int group = p.heads / p.kv_heads, qtiles = (lq + kRows - 1) / kRows, from = max(j - (lk - lq), 0);  // the first query that sees it
    const int most = min(__reduce_max_sync(0xffffffffu, odd ? from : 0), lq);
    const int64_t st = want_v ? p.do_st : p.q_st, sh = want_v ? p.do_sh : p.q_sh;
    const T* x0 = static_cast<const T*>(want_v ? p.dout : p.q) + q0 * st;
    // seen: a row of weights that are not finite makes all of the key so
    auto rows_explain = [&] {
        for (int it = i1 - 1; it >= i0; --it) {
            const int head = kvh * group + it / qtiles, first = (it % qtiles) * kRows;
            const float *lse = p.lse + static_cast<int64_t>(head) * p.tq + q0, *delta = p.delta + static_cast<int64_t>(head) * p.tq + q0;
            for (int i = min(first + kRows, lq) - 1; i >= max(first, from); --i)
                if (!is_finite(lse[i]) || (!want_v && !is_finite(delta[i]))) return true;
        }
        return false;
    };
    bool again = false, explained = false, asked = false;
    for (int it = i0; it < i1; ++it) {
        const int first = (it % qtiles) * kRows, end = min(min(first + kRows, lq), most);
        if (it % qtiles < qt0 || first >= end) continue;
        const T* x = x0 + (kvh * group + it / qtiles) * sh;
        // hidden: rows of the tile before `from`
        const bool some = last_not_finite<T>(x, st, first, end, p.dim) >= 0;
        if (!some || !odd || again || explained) continue;
        if (!asked) explained = rows_explain(), asked = true;
        if (explained) continue;
        const int h1 = min(end, from);
        for (int c = 0; c < p.dim && !again; ++c) {
            bool hidden = false, seen = false;
            for (int r = first; r < h1 && !hidden; ++r) hidden = !is_finite(to_f(x[r * st + c]));
            if (!hidden) continue;
            for (int k = i1 - 1; k >= i0 && !seen; --k) {
                const T* y = x0 + (kvh * group + k / qtiles) * sh;
                const int f = (k % qtiles) * kRows;
                for (int r = min(f + kRows, lq) - 1; r >= max(f, from) && !seen; --r) seen = !is_finite(to_f(y[r * st + c]));
            }
            again = !seen;
        }
    }
    return again;
}

// dk (want_v: dv) of key k, the j-th of its window, over the query tiles [i0, i1) of its heads.
template <typename T>
__device__ __noinline__ void key_row(const AttnParams& p, int64_t k, int j, int kvh, int64_t q0, int lq, int lk, int i0, int i1, float up,
                                     bool want_v, int z) {
    const int64_t row = (k * p.kv_heads + kvh) * p.dim;
    T* out = static_cast<T*>(want_v ? p.dv : p.dk) + row;
    float* part = p.qsplits > 1 ? (want_v ? p.part_dv : p.part_dk) + static_cast<int64_t>(z) * p.tk * p.kv_heads * p.dim + row : nullptr;
    float o[kMaxHeadDim];
    const int group = p.heads / p.kv_heads, qtiles = (lq + kRows - 1) / kRows;
    for (int c = 0; c < kMaxHeadDim; ++c) o[c] = 0.0f;
    for (int it = i0; it < i1; ++it) {
        const int head = kvh * group + it / qtiles, first = (it % qtiles) * kRows;
        for (int i = max(first, j - (lk - lq)); i < min(first + kRows, lq); ++i) {
            const int64_t q = q0 + i;
            const int64_t at = static_cast<int64_t>(head) * p.tq + q;
            float w = ex2(score_of<T>(p, q, k, head, kvh) - p.lse[at]) * far_factor(p, at, p.lse[at]);
            const T* g = static_cast<const T*>(p.dout) + q * p.do_st + head * p.do_sh;
            const T* with = g;
            if (!want_v) {
                w *= (dot_row(g, static_cast<const T*>(p.v) + k * p.v_st + kvh * p.v_sh, p.dim) -
                      p.delta[at]) * up;
                with = static_cast<const T*>(p.q) + q * p.q_st + head * p.q_sh;
            }
            w = to_f(from_f<T>(w));
            for (int c = 0; c < p.dim; ++c) o[c] = fmaf(w, to_f(with[c]), o[c]);
        }
    }
    const float by = want_v ? 1.0f : p.scale / up;
    for (int c = 0; c < p.dim; ++c) {
        if (part != nullptr)
            part[c] = o[c] * by;
        else
            out[c] = from_f<T>(o[c] * by);
    }
}

// A row of dk or dv out of tensor memory. Whole warps; rows of lanes with `live`. `staged`: to row r of the panel at
// `to` instead of memory. True: some value is not finite, in a causal window.
template <typename T, int DP>
__device__ __forceinline__ bool finish_key_row(const AttnParams& p, uint32_t at, bool live, bool any, int64_t k, int kvh, int z,
                                               float up, bool want_v, bool alive, bool staged, uint32_t to, int r) {
    const int64_t row = (k * p.kv_heads + kvh) * p.dim;
    T* out = static_cast<T*>(want_v ? p.dv : p.dk) + row;
    float* part = p.qsplits > 1 ? (want_v ? p.part_dv : p.part_dk) + static_cast<int64_t>(z) * p.tk * p.kv_heads * p.dim + row : nullptr;
    const float by = !alive ? kNaN : want_v ? 1.0f : p.scale / up;
    bool fine = true;
#pragma unroll
    for (int c = 0; c < DP; c += 16) {
        if (c >= p.dim) continue;
        float o[16];
        if (any) {
            tc::tmem_ld16(at + c, o);
            tc::wait_ld();
        } else {
#pragma unroll
            for (int i = 0; i < 16; ++i) o[i] = 0.0f;
        }
#pragma unroll
        for (int i = 0; i < 16; ++i) fine = fine && is_finite(o[i]);
        if (!live) continue;
        if (part != nullptr) {
#pragma unroll
            for (int i = 0; i < 16; ++i) o[i] *= by;
            write_part(part, o, c, p.dim);
        } else if (staged) {
            stage16<T>(to, r, o, c, by);
        } else {
            write_out<T>(out, o, c, p.dim, by);
        }
    }
    return p.causal && live && !fine && alive;
}

// ---- which windows there are -----------------------------------------------------------------
__global__ void __launch_bounds__(256) k_attn_flags(AttnParams p, int* flags) {
    int some = 0;
    for (int w = blockIdx.x * 256 + threadIdx.x; w < p.windows; w += gridDim.x * 256) {
        const int n = attn_offset(p.k_off, p.windows, p.tk, w + 2) - attn_offset(p.k_off, p.windows, p.tk, w + 1);
        some |= n > p.short_max ? kSomeLong : n > p.tiny_max ? kSomeShort : 0;
    }
    some = __reduce_or_sync(0xffffffffu, some);
    if (some != 0 && (threadIdx.x & 31) == 0) atomicOr(flags, some);
}

// The same, with the windows of the warp-level kernels listed in order: a block, 1024 windows at a time.
__global__ void __launch_bounds__(1024) k_attn_lists(AttnParams p, int* flags) {
    __shared__ int sums[2][32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int some = 0, base[2] = {0, 0};
    for (int w0 = 0; w0 < p.windows; w0 += 1024) {
        const int w = w0 + threadIdx.x;
        int cls = -1;
        if (w < p.windows) {
            const int n = attn_offset(p.k_off, p.windows, p.tk, w + 2) - attn_offset(p.k_off, p.windows, p.tk, w + 1);
            some |= n > p.short_max ? kSomeLong : n > p.tiny_max ? kSomeShort : 0;
            if (n > 0 && n <= p.tiny_max) cls = n <= 16 ? 0 : 1;
        }
        const unsigned in[2] = {__ballot_sync(0xffffffffu, cls == 0), __ballot_sync(0xffffffffu, cls == 1)};
        if (lane < 2) sums[lane][warp] = __popc(lane == 0 ? in[0] : in[1]);
        __syncthreads();
#pragma unroll
        for (int c = 0; c < 2; ++c) {
            int before = base[c], all = 0;
            for (int k = 0; k < 32; ++k) {
                if (k == warp) before += all;
                all += sums[c][k];
            }
            if (cls == c) p.tiny_list[c * p.windows + before + __popc(in[c] & ((1u << lane) - 1u))] = w;
            base[c] += all;
        }
        __syncthreads();
    }
    some = __reduce_or_sync(0xffffffffu, some);
    if (some != 0 && lane == 0) atomicOr(flags, some);
    if (threadIdx.x < 2) flags[1 + threadIdx.x] = base[threadIdx.x];
}

// The largest finite |dout| and |v| of each window and key head, fp16. A block takes 128 rows of a window's
// queries, or of its keys; its warps share out key heads and rows, eight lanes a row. 34560 queries and
// 77760 keys of 6 heads of 30: 18 us (38 us with the loads of one row at a time on their way).
__global__ void __launch_bounds__(256) k_attn_window_max(const __grid_constant__ AttnParams p, int q_slots) {
    const bool of_q = static_cast<int>(blockIdx.x) < q_slots;
    AttnTile t;
    if (!attn_tile(of_q ? p.q_off : p.k_off, of_q ? p.tq : p.tk, of_q ? p.k_off : p.q_off, of_q ? p.tk : p.tq, p.windows, 1, kRows,
                   of_q ? blockIdx.x : blockIdx.x - q_slots, t))
        return;
    if (t.window < 0 || t.olen == 0) return;
    const int group = of_q ? p.heads / p.kv_heads : 1, rows = min(kRows, t.len - t.first), lane = threadIdx.x & 31;
    const int64_t st = of_q ? p.do_st : p.v_st, sh = of_q ? p.do_sh : p.v_sh;
    const unsigned short* base = static_cast<const unsigned short*>(of_q ? p.dout : p.v) + (static_cast<int64_t>(t.begin) + t.first) * st;
    const uintptr_t at = reinterpret_cast<uintptr_t>(base);
    const bool vec = ((at & 15) | ((st | sh | p.dim) & 7)) == 0, pairs = ((at & 3) | ((st | sh | p.dim) & 1)) == 0;
    const int parts = p.kv_heads < 8 ? 8 / p.kv_heads : 1;
    auto of = [](uint32_t x) {  // of two values
        const uint32_t a = x & 0x7fffu, b = (x >> 16) & 0x7fffu;
        return max(a < 0x7c00u ? a : 0u, b < 0x7c00u ? b : 0u);
    };
    for (int unit = threadIdx.x >> 5; unit < p.kv_heads * parts; unit += 8) {
        const int kvh = unit % p.kv_heads;
        uint32_t m = 0u;
        const int r0 = unit / p.kv_heads * 4 + (lane >> 3), step = 4 * parts;
        for (int g = 0; g < group; ++g) {
            const unsigned short* head = base + (kvh * group + g) * sh;
            // column by column of a lane, so that the loads of eight rows are on their way together
            if (vec) {
                for (int c = 8 * (lane & 7); c < p.dim; c += 64)
#pragma unroll 8
                    for (int r = r0; r < rows; r += step) {
                        const uint4 x = __ldg(reinterpret_cast<const uint4*>(head + r * st + c));
                        m = max(m, max(max(of(x.x), of(x.y)), max(of(x.z), of(x.w))));
                    }
            } else if (pairs) {
                for (int c = 2 * (lane & 7); c < p.dim; c += 16)
#pragma unroll 8
                    for (int r = r0; r < rows; r += step) m = max(m, of(__ldg(reinterpret_cast<const uint32_t*>(head + r * st + c))));
            } else {
                for (int c = lane & 7; c < p.dim; c += 8)
#pragma unroll 8
                    for (int r = r0; r < rows; r += step) m = max(m, of(__ldg(head + r * st + c)));
            }
        }
        m = __reduce_max_sync(0xffffffffu, m);
        if (lane == 0 && m != 0u) atomicMax(p.win_max + (static_cast<int64_t>(t.window) * p.kv_heads + kvh) * 2 + (of_q ? 0 : 1), m);
    }
}

// ---- short windows ---------------------------------------------------------------------------
template <int DP>
struct ShortSmem {
    static constexpr int kT = kRows * DP * 2, kK = kShortKeys * DP * 2, kP = kRows * kShortKeys * 2;
    // dS, P, Q, dO, K, V; dS and P end before 16 KB that may be read past them (rows of keys 64 and on,
    // which nothing uses)
    static constexpr int kTiles = 2 * kP + 2 * kT + 2 * kK;
    static constexpr int kBytes = kTiles + static_cast<int>(sizeof(KeyPos<kShortKeys>)) + 64 + 128 + 2 * kRows * 4;
};

template <typename T, int DP, bool BIAS>
__global__ void __launch_bounds__(2 * kRows, DP == 64 ? 2 : 1) k_attn_bwd_short(const __grid_constant__ AttnParams p) {
    using L = ShortSmem<DP>;
    constexpr int kCols = DP == 64 ? 256 : 512, KT = kShortKeys, kThreads = 2 * kRows, N = KT / 2;
    extern __shared__ __align__(16) unsigned char smem_raw[];
    unsigned char* base = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    const uint32_t sd = tc::smem_addr(base), sp = sd + L::kP, sq = sp + L::kP, sg = sq + L::kT, sk = sg + L::kT, sv = sk + L::kK;
    KeyPos<KT>* kp = reinterpret_cast<KeyPos<KT>*>(base + L::kTiles);
    Range* qrange = reinterpret_cast<Range*>(kp + 1);
    uint64_t* bars = reinterpret_cast<uint64_t*>(qrange + 4);
    uint32_t* slot_tmem = reinterpret_cast<uint32_t*>(bars + 2);
    volatile int* dead = reinterpret_cast<volatile int*>(slot_tmem + 1);
    float* wsize = reinterpret_cast<float*>(bars + 4);
    float* wsum = wsize + 8;
    float* half_delta = reinterpret_cast<float*>(bars + 16);  // [2][kRows]
    const int group = p.heads / p.kv_heads, entries = BIAS ? bias_entries(p.bias) : 0, kvh = blockIdx.y;
    const bool grad_bias = BIAS && p.bias_part != nullptr;
    double* acc = reinterpret_cast<double*>(base + L::kBytes);
    int* I = reinterpret_cast<int*>(acc + (grad_bias ? group * entries : 0));
    float* E = reinterpret_cast<float*>(I + (grad_bias ? entries : 0));
    const uint32_t bar_s = tc::smem_addr(bars), bar_o = bar_s + 8, bar_end = bar_s + 24;

    const int tid = threadIdx.x, warp = tid >> 5, row = tid & (kRows - 1), j0 = (tid / kRows) * N, z = blockIdx.z;
    const int dim16 = (p.dim + 15) & ~15;
    const Loader<T, kThreads> ok(p.k, p.k_st, p.k_sh, p.dim, kvh), ov(p.v, p.v_st, p.v_sh, p.dim, kvh),
        oq(p.q, p.q_st, p.q_sh, p.dim, kvh * group), og(p.dout, p.do_st, p.do_sh, p.dim, kvh * group);
    // rows outside every window
    if (z == 0) {
        const int q_lo = attn_offset(p.q_off, p.windows, p.tq, 1), q_hi = attn_offset(p.q_off, p.windows, p.tq, p.windows + 1);
        const int k_lo = attn_offset(p.k_off, p.windows, p.tk, 1), k_hi = attn_offset(p.k_off, p.windows, p.tk, p.windows + 1);
        const int nq = q_lo + max(p.tq - q_hi, 0), nk = k_lo + max(p.tk - k_hi, 0);
        for (int r = blockIdx.x; r < nq + nk; r += gridDim.x) {
            const bool of_q = r < nq;
            const int i = of_q ? r : r - nq, lo = of_q ? q_lo : k_lo, hi = of_q ? q_hi : k_hi;
            const int64_t token = i < lo ? i : hi + (i - lo);
            for (int c = tid; c < p.dim * (of_q ? group : 2); c += kThreads) {
                if (of_q) {
                    static_cast<T*>(p.dq)[(token * p.heads + kvh * group) * p.dim + c] = from_f<T>(0.0f);
                } else if (p.qsplits == 1) {
                    static_cast<T*>(c < p.dim ? p.dk : p.dv)[(token * p.kv_heads + kvh) * p.dim + c % p.dim] = from_f<T>(0.0f);
                } else {
                    for (int s = 0; s < p.qsplits; ++s)
                        (c < p.dim ? p.part_dk : p.part_dv)[((static_cast<int64_t>(s) * p.tk + token) * p.kv_heads + kvh) * p.dim + c % p.dim] = 0.0f;
                }
            }
        }
    }

    // and windows without keys
    if (z == 0)
        for (int w = blockIdx.x; w < p.windows; w += gridDim.x) {
            const int q0 = attn_offset(p.q_off, p.windows, p.tq, w + 1), lq = attn_offset(p.q_off, p.windows, p.tq, w + 2) - q0;
            if (attn_offset(p.k_off, p.windows, p.tk, w + 2) > attn_offset(p.k_off, p.windows, p.tk, w + 1)) continue;
            const int per = group * p.dim;
            for (int64_t i = tid; i < static_cast<int64_t>(lq) * per; i += kThreads)
                static_cast<T*>(p.dq)[((q0 + i / per) * p.heads + kvh * group) * p.dim + i % per] = from_f<T>(0.0f);
        }
    if ((*p.flags & kSomeShort) == 0) return;

    if (tid == 0) {
        tc::mbar_init(bar_s, 1);
        tc::mbar_init(bar_o, 1);
        tc::mbar_init(bar_end, 1);
        tc::mbar_init_fence();
        *dead = 0;
    }
    if (warp == 0) tc::tmem_alloc<kCols>(tc::smem_addr(slot_tmem));
    if constexpr (BIAS)
    for (int e = tid; e < entries * group; e += kThreads) {
        E[e] = bias_entry(p.bias, p.heads, kvh * group + e / entries, e % entries);
        if (grad_bias) acc[e] = 0.0;
    }
    if (grad_bias)
        for (int e = tid; e < entries; e += kThreads) I[e] = 0;
    tc::fence_before();
    __syncthreads();
    tc::fence_after();
    const uint32_t tmem = *slot_tmem, ts = tmem + (static_cast<uint32_t>((warp & 3) * 32) << 16);
    const uint32_t t_dv = 2 * KT, t_dk = 2 * KT + DP;  // columns; S at 0, dP at 64, dQ over both
    const uint32_t id_grad = tc::idesc(kIsBf16<T>, dim16, true, true), id_q = tc::idesc(kIsBf16<T>, dim16, false, true);
    int par_s = 0, par_o = 0;
    bool alive = true;

    for (int w = blockIdx.x; w < p.windows; w += gridDim.x) {
        const int q0 = attn_offset(p.q_off, p.windows, p.tq, w + 1), lq = max(attn_offset(p.q_off, p.windows, p.tq, w + 2) - q0, 0);
        const int k0 = attn_offset(p.k_off, p.windows, p.tk, w + 1), lk = max(attn_offset(p.k_off, p.windows, p.tk, w + 2) - k0, 0);
        if (lk > p.short_max || lk <= p.tiny_max) continue;  // other kernels', and windows without keys
        const float up = ds_scale<T>(p, w, kvh);
        const int qtiles = (lq + kRows - 1) / kRows, total = group * qtiles, per = (total + p.qsplits - 1) / p.qsplits;
        const int i0 = min(z * per, total), i1 = min(i0 + per, total);
        const int n = lk, n16 = (n + 15) & ~15;
        float lse = INFINITY, far = 1.0f;
        int2 qp = make_int2(0, 0);
        // Q, dO and the row's scalars of one tile
        auto fetch = [&](int it) {
            const int head = kvh * group + it / qtiles, first = (it % qtiles) * kRows, rows = min(kRows, lq - first);
            oq.load(sq, kRows, q0 + first, rows, kRows, (it / qtiles) * p.q_sh);
            og.load(sg, kRows, q0 + first, rows, kRows, (it / qtiles) * p.do_sh);
            tc::cp_async_commit();
            const int64_t at = static_cast<int64_t>(head) * p.tq + q0 + first + min(row, rows - 1);
            lse = row < rows ? p.lse[at] : INFINITY;
            far = far_factor(p, at, lse);
            if (BIAS) qp = bias_pos(p.bias.q_pos, p.bias.axes, q0 + first + min(row, rows - 1));
        };
        __syncthreads();  // the window before has read its keys
        if (i0 < i1) {
            ok.load(sk, KT, k0, n, n16);
            ov.load(sv, KT, k0, n, n16);
            fetch(i0);
            if (BIAS) load_key_pos<KT>(kp, p.bias, k0, n);
        }
        for (int it = i0; it < i1; ++it) {
            const int g = it / qtiles, head = kvh * group + g, first = (it % qtiles) * kRows, rows = min(kRows, lq - first);
            if (BIAS) {
                const Range r = warp_range(qp);
                if (tid < kRows && (tid & 31) == 0) qrange[warp] = r;
            }
            tc::cp_async_wait<0>();
            tc::fence_async();
            tc::fence_before();
            if (__syncthreads_or(!alive)) {  // a wait has run out: nothing more is issued, the rows become NaN
                alive = false;
                for (int i = tid; i < rows * p.dim; i += kThreads)
                    static_cast<T*>(p.dq)[(static_cast<int64_t>(q0 + first + i / p.dim) * p.heads + head) * p.dim + i % p.dim] = from_f<T>(kNaN);
                continue;
            }
            if (warp == 0 && tc::elect_one()) {
                tc::fence_after();
                const uint32_t id = tc::idesc(kIsBf16<T>, n16, false, false);
                tc::mma_nt<DP, kRows, KT>(tmem, sq, sk, dim16, id);
                tc::mma_nt<DP, kRows, KT>(tmem + KT, sg, sv, dim16, id);
                tc::commit(bar_s);
            }
            const int see = row >= rows ? 0 : p.causal ? min(max(first + row + lk - lq + 1, 0), lk) : lk;
            const bool whole = n == n16 && (!p.causal || first + lk - lq + 1 >= n);
            BiasMode mode = kOne;
            if (BIAS) mode = bias_mode(p.bias, join(join(qrange[0], qrange[1]), join(qrange[2], qrange[3])), key_range(kp));
            alive = tc::mbar_wait(bar_s, par_s, dead) && alive;
            par_s ^= 1;
            tc::fence_after();
            float s[N], dp[N];
            weights<KT, BIAS>(p, s, dp, ts, ts + KT, n16, j0, whole, see, lse, far, mode, E + g * entries, kp, qp);
            float2 d0 = make_float2(0.0f, 0.0f), d1 = d0;
#pragma unroll
            for (int c = 0; c < N; c += 4) {
                d0 = __ffma2_rn(make_float2(s[c], s[c + 1]), make_float2(dp[c], dp[c + 1]), d0);
                d1 = __ffma2_rn(make_float2(s[c + 2], s[c + 3]), make_float2(dp[c + 2], dp[c + 3]), d1);
            }
            half_delta[tid] = (d0.x + d0.y) + (d1.x + d1.y);
            write_row<T>(sp, row, j0, s, 1.0f);
            __syncthreads();  // the other half of the row's keys
            const float delta = half_delta[row] + half_delta[kRows + row];
            score_gradients(s, dp, delta, j0, whole, see);
            write_row<T>(sd, row, j0, dp, up);
            if (grad_bias) {
                const float m = warp_size(dp);
                if ((tid & 31) == 0) wsize[warp] = m;
            }
            if (p.causal && tid < rows) p.delta[static_cast<int64_t>(head) * p.tq + q0 + first + tid] = delta;  // tid: one of the two
            tc::fence_async();
            tc::fence_before();
            if (__syncthreads_or(!alive)) alive = false;  // two threads share a row
            if (alive && warp == 0 && tc::elect_one()) {
                tc::fence_after();
                tc::mma_tt<kRows>(tmem + t_dv, tc::desc(sp, L::kP), tc::desc(sg, kRows * 128), id_grad, it > i0);
                tc::mma_tt<kRows>(tmem + t_dk, tc::desc(sd, L::kP), tc::desc(sq, kRows * 128), id_grad, it > i0);
                const uint64_t dd = tc::desc(sd, 16), dk = tc::desc(sk, KT * 128);
#pragma unroll
                for (int k = 0; k < KT; k += 16)
                    if (k < n16) tc::mma_ss(tmem, dd + k * 2 / 16, dk + k * 128 / 16, id_q, k > 0);
                tc::commit(bar_o);
            }
            BiasSum bs{kOne, 0.0f, false};
            if (grad_bias) {
                bs = bias_sum<8>(mode, wsize);
                if (bs.fixed != 0.0f || bs.bad) bias_add<KT>(p, bs, dp, n16, head, kp, j0, qp, I, wsum + warp);
            }
            alive = tc::mbar_wait(bar_o, par_o, dead) && alive;
            par_o ^= 1;
            tc::fence_after();
            const int2 qp_now = qp;
            const float lse_now = lse, far_now = far;
            if (it + 1 < i1) fetch(it + 1);
            // columns of dQ in turn between the two threads of a row
            bool fine = true;
#pragma unroll
            for (int c = 0; c < DP; c += 16) {
                if (c >= dim16 || ((c >> 4) & 1) != tid / kRows) continue;
                float o[16];
                tc::tmem_ld16(ts + c, o);
                tc::wait_ld();
#pragma unroll
                for (int i = 0; i < 16; ++i) fine = fine && is_finite(o[i]);
                stage16<T>(sd, row, o, c, alive ? p.scale / up : kNaN);
            }
            if (p.causal) {
                if (__syncthreads_or(!fine)) {  // some row of the tile: whoever holds one of its threads
                    half_delta[tid] = fine ? 0.0f : 1.0f;
                    __syncthreads();
                    const bool odd = row < rows && half_delta[row] + half_delta[kRows + row] != 0.0f && alive;
                    if (tid < kRows && query_again<T>(p, odd, k0, kvh, see, n, lse_now, delta))
                        query_row<T>(p, q0 + first + tid, head, k0, see, lse_now, far_now, delta, up, sd);
                }
            }
            tc::fence_before();
            __syncthreads();
            if (grad_bias && (bs.fixed != 0.0f || bs.bad))
                bias_join<kThreads, 8, KT>(p, bs, entries, head, kp, qp_now, I, wsum, acc + g * entries);
            store_panel<T, kThreads>(sd, p.dq, p.heads, p.dim, q0, head, 1, first, rows);
        }
        if (__syncthreads_or(!alive)) alive = false;  // one thread's weights are in every row
        if ((warp & 3) < 2) {
            const bool of_v = tid < kRows;
            const int64_t key = k0 + min(row, n - 1);
            const bool odd = finish_key_row<T, DP>(p, ts + (of_v ? t_dv : t_dk), row < n, i0 < i1, key, kvh, z, up, of_v, alive, false, 0, 0);
            if (p.causal && key_again<T>(p, odd, row, kvh, q0, lq, lk, 0, i0, i1, of_v))
                key_row<T>(p, key, row, kvh, q0, lq, lk, i0, i1, up, of_v, z);
        }
        tc::fence_before();
    }
    const bool lost = __syncthreads_or(!alive);
    if constexpr (BIAS) if (grad_bias) {
        for (int e = tid; e < entries * group; e += kThreads)
            p.bias_part[(static_cast<int64_t>(kvh * group + e / entries) * p.bias_parts + p.bias_tiny + z * gridDim.x + blockIdx.x) * entries +
                        e % entries] = lost ? kNaN : acc[e];
    }
    tc::fence_before();
    finish_block(lost, bar_end);
    if (warp == 0) tc::tmem_free<kCols>(tmem);
}

// The tiles of a block: an even range of slots, whose empty ones even out. (Dealt back and forth over the blocks by
// number, so that each gets first and last tiles of causal windows, one window of 16320, 8 heads of 64, forward and
// backward took 4.55 ms against 3.93, two of 4096 and 16 heads 1.32 against 1.30, seven of 4095 down to 1 token 1.17
// against 1.17; one of 8192 and 32 heads 4.13 against 4.24, six of 3000 down to 11 tokens 0.74 against 0.85.)
template <int ROWS>
__device__ __forceinline__ bool walk_range(AttnWalk<ROWS>& walk, int slots, const AttnParams& p, const int32_t* off, int t, const int32_t* other, int ot) {
    const int64_t n = slots;
    return walk.start(off, t, other, ot, p.windows, 1, static_cast<int>(n * blockIdx.x / gridDim.x),
                      static_cast<int>(n * (blockIdx.x + 1) / gridDim.x));
}

// ---- long windows: dq ------------------------------------------------------------------------
// dq: with up to 64 columns 64 keys a tile and two blocks on an SM, which fill each other's waits;
// with more, tensor memory holds one block, of 512 threads. 135 windows of 256 under 576, 6 heads of 30, with
// the bias gradient: 384 us; latency at 24% of an SM's warps, with half of the issue slots and of shared memory's pipe
// taken by the softmax's arithmetic and the bias's sums, and 3% of the tensor pipe.
template <int DP>
struct DqShape {
    static constexpr int KT = DP == 64 ? 64 : 128, kThreads = 4 * KT, N = 32;
    static constexpr int kBuf = DP == 64 ? 2 : 1;  // of the keys and values
    static constexpr int kT = kRows * DP * 2, kK = KT * DP * 2, kP = kRows * KT * 2;
    static constexpr int kTiles = 2 * kT + 2 * kBuf * kK + kP;
    static constexpr int kBytes = kTiles + static_cast<int>(sizeof(KeyPos<KT>)) * kBuf + 64 + 64 + 128;
    static constexpr int kCols = DP == 64 ? 256 : 512;  // S, dP, dQ
};
// dk, dv: the same. Products of 64 keys leave half of their 128 rows unused, but two blocks fill each other's
// waits: 413 us for those windows, against 596 us with 128 keys and one block of 512 threads, and 486 us when
// that had three buffers of queries and one barrier a step.
template <int DP>
struct DkvShape {
    static constexpr int KT = DP == 64 ? 64 : 128, kThreads = 4 * KT, N = 32;
    static constexpr int kT = kRows * DP * 2, kK = KT * DP * 2, kP = kRows * KT * 2;
    static constexpr int kTiles = 2 * kP + 2 * kT + 2 * kK;
    static constexpr int kBytes = kTiles + static_cast<int>(sizeof(KeyPos<KT>)) + 8 * static_cast<int>(sizeof(Range)) + 64;
    static constexpr int kCols = DP == 64 ? 256 : 512;  // S, dP, dV, dK
};

template <typename T, int DP, bool BIAS>
__global__ void __launch_bounds__(DqShape<DP>::kThreads, DP == 64 ? 2 : 1) k_attn_dq_long(const __grid_constant__ AttnParams p) {
    if ((*p.flags & kSomeLong) == 0) return;
    using L = DqShape<DP>;
    constexpr int KT = L::KT, kBuf = L::kBuf, kThreads = L::kThreads, N = L::N, kWarps = kThreads / 32;
    extern __shared__ __align__(16) unsigned char smem_raw[];
    unsigned char* base = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    const uint32_t sq = tc::smem_addr(base), sg = sq + L::kT, sk = sg + L::kT, sv = sk + kBuf * L::kK, sd = sv + kBuf * L::kK;
    KeyPos<KT>* kps = reinterpret_cast<KeyPos<KT>*>(base + L::kTiles);
    Range* qrange = reinterpret_cast<Range*>(kps + kBuf);
    uint64_t* bars = reinterpret_cast<uint64_t*>(qrange + 4);
    uint32_t* slot_tmem = reinterpret_cast<uint32_t*>(bars + 2);
    volatile int* dead = reinterpret_cast<volatile int*>(slot_tmem + 1);
    float* wsize = reinterpret_cast<float*>(bars + 8);
    float* wsum = wsize + 16;
    const int entries = BIAS ? bias_entries(p.bias) : 0, head = blockIdx.y, kvh = head / (p.heads / p.kv_heads);
    const bool grad_bias = BIAS && p.bias_part != nullptr;
    double* acc = reinterpret_cast<double*>(base + L::kBytes);
    int* I = reinterpret_cast<int*>(acc + (grad_bias ? entries : 0));
    float* E = reinterpret_cast<float*>(I + (grad_bias ? entries : 0));
    const uint32_t bar_s = tc::smem_addr(bars), bar_o = bar_s + 8, bar_end = bar_s + 24;

    const int tid = threadIdx.x, warp = tid >> 5, row = tid & (kRows - 1), j0 = (tid / kRows) * N;
    const int dim16 = (p.dim + 15) & ~15, slots = attn_slots(p.tq, p.windows, kRows);
    const Loader<T, kThreads> ok(p.k, p.k_st, p.k_sh, p.dim, kvh), ov(p.v, p.v_st, p.v_sh, p.dim, kvh),
        oq(p.q, p.q_st, p.q_sh, p.dim, head), og(p.dout, p.do_st, p.do_sh, p.dim, head);
    if (tid == 0) {
        tc::mbar_init(bar_s, 1);
        tc::mbar_init(bar_o, 1);
        tc::mbar_init(bar_end, 1);
        tc::mbar_init_fence();
        *dead = 0;
    }
    if (warp == 0) tc::tmem_alloc<L::kCols>(tc::smem_addr(slot_tmem));
    for (int e = tid; e < entries; e += kThreads) {
        E[e] = bias_entry(p.bias, p.heads, head, e);
        if (grad_bias) acc[e] = 0.0, I[e] = 0;
    }
    tc::fence_before();
    __syncthreads();
    tc::fence_after();
    const uint32_t tmem = *slot_tmem, ts = tmem + (static_cast<uint32_t>((warp & 3) * 32) << 16);
    const uint32_t id_q = tc::idesc(kIsBf16<T>, dim16, false, true);
    int par_s = 0, par_o = 0;
    bool alive = true;

    AttnWalk<kRows> walk;
    for (bool more = walk_range(walk, slots, p, p.q_off, p.tq, p.k_off, p.tk); more; more = walk.next()) {
        const AttnTile& t = walk.tile;
        if (t.window < 0 || t.olen <= p.short_max) continue;
        const float up = ds_scale<T>(p, t.window, kvh);
        const int rows = min(kRows, t.len - t.first), shift = t.olen - t.len;
        const bool live = row < rows;
        const int see = !live ? 0 : p.causal ? min(max(t.first + row + shift + 1, 0), t.olen) : t.olen;
        const int most = p.causal ? min(max(t.first + rows + shift, 0), t.olen) : t.olen;
        const int least = p.causal ? min(max(t.first + shift + 1, 0), t.olen) : t.olen;
        const int tiles = (most + KT - 1) / KT;
        const int64_t token = t.begin + t.first + min(row, rows - 1);
        const float lse = live ? p.lse[static_cast<int64_t>(head) * p.tq + token] : INFINITY;
        const float far = far_factor(p, static_cast<int64_t>(head) * p.tq + token, lse);
        const float delta = live ? p.delta[static_cast<int64_t>(head) * p.tq + token] : 0.0f;
        const int2 qp = entries > 0 ? bias_pos(p.bias.q_pos, p.bias.axes, token) : make_int2(0, 0);
        auto fetch = [&](int kt) {
            const int b = kBuf == 2 ? kt & 1 : 0, n = min(KT, most - kt * KT), n16 = (n + 15) & ~15;
            ok.load(sk + b * L::kK, KT, t.obegin + kt * KT, n, n16);
            ov.load(sv + b * L::kK, KT, t.obegin + kt * KT, n, n16);
            if (BIAS) load_key_pos<KT>(kps + b, p.bias, t.obegin + kt * KT, n);
        };
        __syncthreads();  // the tile before has been read
        if (tiles > 0) {
            oq.load(sq, kRows, t.begin + t.first, rows, kRows);
            og.load(sg, kRows, t.begin + t.first, rows, kRows);
            fetch(0);
            if (BIAS) {
                const Range r = warp_range(qp);
                if (tid < kRows && (tid & 31) == 0) qrange[warp] = r;
            }
        }
        tc::cp_async_commit();
        BiasSum bs{kOne, 0.0f, false};
        for (int kt = 0; kt < tiles; ++kt) {
            const int b = kBuf == 2 ? kt & 1 : 0, n = min(KT, most - kt * KT), n16 = (n + 15) & ~15;
            KeyPos<KT>* kp = kps + b;
            tc::cp_async_wait<0>();
            tc::fence_async();
            tc::fence_before();
            if (__syncthreads_or(!alive)) {  // a wait has run out: nothing more is issued
                alive = false;
                break;
            }
            if (warp == 0 && tc::elect_one()) {
                tc::fence_after();
                const uint32_t id = tc::idesc(kIsBf16<T>, n16, false, false);
                tc::mma_nt<DP, kRows, KT>(tmem, sq, sk + b * L::kK, dim16, id);
                tc::mma_nt<DP, kRows, KT>(tmem + KT, sg, sv + b * L::kK, dim16, id);
                tc::commit(bar_s);
            }
            if (grad_bias && kt > 0 && (bs.fixed != 0.0f || bs.bad))  // of the tile before
                bias_join<kThreads, kWarps, KT>(p, bs, entries, head, kps + (kBuf == 2 ? (kt - 1) & 1 : 0), qp, I, wsum, acc);
            if (kBuf == 2) {
                if (kt > 0) {  // dQ of the tile before: its keys and dS are free
                    alive = tc::mbar_wait(bar_o, par_o, dead) && alive;
                    par_o ^= 1;
                }
                if (grad_bias) __syncthreads();  // its key positions have been read
                if (kt + 1 < tiles) fetch(kt + 1);
                tc::cp_async_commit();
            }
            BiasMode mode = kOne;
            if (BIAS) mode = bias_mode(p.bias, join(join(qrange[0], qrange[1]), join(qrange[2], qrange[3])), key_range(kp));
            alive = tc::mbar_wait(bar_s, par_s, dead) && alive;
            par_s ^= 1;
            tc::fence_after();
            float s[N], dp[N];
            const bool whole = n == n16 && kt * KT + n <= least;
            weights<KT, BIAS>(p, s, dp, ts, ts + KT, n16, j0, whole, see - kt * KT, lse, far, mode, E, kp, qp);
            score_gradients(s, dp, delta, j0, whole, see - kt * KT);
            write_row<T>(sd, row, j0, dp, up);
            if (grad_bias) {
                const float m = warp_size(dp);
                if ((tid & 31) == 0) wsize[warp] = m;
            }
            tc::fence_async();
            tc::fence_before();
            __syncthreads();
            if (warp == 0 && tc::elect_one()) {
                tc::fence_after();
                const uint64_t dd = tc::desc(sd, 16), dk = tc::desc(sk + b * L::kK, KT * 128);
#pragma unroll
                for (int k = 0; k < KT; k += 16)
                    if (k < n16)
                        tc::mma_ss(tmem + 2 * KT, dd + ((k >> 6) * kRows * 128 + (k & 63) * 2) / 16, dk + k * 128 / 16, id_q, kt > 0 || k > 0);
                tc::commit(bar_o);
            }
            if (grad_bias) {
                bs = bias_sum<kWarps>(mode, wsize);
                if (bs.fixed != 0.0f || bs.bad) bias_add<KT>(p, bs, dp, n16, head, kp, j0, qp, I, wsum + warp);
            }
            if (kBuf == 1) {
                alive = tc::mbar_wait(bar_o, par_o, dead) && alive;
                par_o ^= 1;
                if (kt + 1 < tiles) {
                    if (grad_bias) {
                        __syncthreads();
                        if (bs.fixed != 0.0f || bs.bad) bias_join<kThreads, kWarps, KT>(p, bs, entries, head, kp, qp, I, wsum, acc);
                        bs = BiasSum{kOne, 0.0f, false};
                        __syncthreads();
                    } else if (BIAS) {
                        __syncthreads();
                    }
                    fetch(kt + 1);
                }
                tc::cp_async_commit();
            }
        }
        if (tiles > 0 && kBuf == 2) {
            alive = tc::mbar_wait(bar_o, par_o, dead) && alive;
            par_o ^= 1;
        }
        tc::fence_after();
        if (__syncthreads_or(!alive)) alive = false;  // one thread's part is in others' rows
        if (grad_bias && tiles > 0 && (bs.fixed != 0.0f || bs.bad))
            bias_join<kThreads, kWarps, KT>(p, bs, entries, head, kps + (kBuf == 2 ? (tiles - 1) & 1 : 0), qp, I, wsum, acc);
        if (tid < kRows) {
            bool fine = true;
#pragma unroll
            for (int c = 0; c < DP; c += 16) {
                if (c >= dim16) continue;
                float o[16];
                if (tiles > 0) {
                    tc::tmem_ld16(ts + 2 * KT + c, o);
                    tc::wait_ld();
                } else {
#pragma unroll
                    for (int i = 0; i < 16; ++i) o[i] = 0.0f;
                }
#pragma unroll
                for (int i = 0; i < 16; ++i) fine = fine && is_finite(o[i]);
                stage16<T>(sq, row, o, c, alive ? p.scale / up : kNaN);
            }
            if (p.causal && query_again<T>(p, live && !fine && alive, t.obegin, kvh, see, most, lse, delta))
                query_row<T>(p, token, head, t.obegin, see, lse, far, delta, up, sq);
        }
        tc::fence_before();
        __syncthreads();
        store_panel<T, kThreads>(sq, p.dq, p.heads, p.dim, t.begin, head, 1, t.first, rows);
    }
    const bool lost = __syncthreads_or(!alive);
    if (grad_bias)
        for (int e = tid; e < entries; e += kThreads)
            p.bias_part[(static_cast<int64_t>(head) * p.bias_parts + p.bias_tiny + p.bias_short + blockIdx.x) * entries + e] = lost ? kNaN : acc[e];
    tc::fence_before();
    finish_block(lost, bar_end);
    if (warp == 0) tc::tmem_free<L::kCols>(tmem);
}

// ---- long windows: dk, dv --------------------------------------------------------------------
template <typename T, int DP, bool BIAS>
__global__ void __launch_bounds__(DkvShape<DP>::kThreads, DP == 64 ? 2 : 1) k_attn_dkv_long(const __grid_constant__ AttnParams p) {
    if ((*p.flags & kSomeLong) == 0) return;
    using L = DkvShape<DP>;
    constexpr int KT = L::KT, kThreads = L::kThreads, N = L::N;
    extern __shared__ __align__(16) unsigned char smem_raw[];
    unsigned char* base = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    // P and dS first: with tiles of 64 keys the products still take 128 of their columns, the second half
    // from what lies behind, for rows of dK and dV that nobody reads
    const uint32_t sp = tc::smem_addr(base), sd = sp + L::kP, sq = sd + L::kP, sg = sq + L::kT, sk = sg + L::kT, sv = sk + L::kK;
    KeyPos<KT>* kp = reinterpret_cast<KeyPos<KT>*>(base + L::kTiles);
    Range* qrange = reinterpret_cast<Range*>(kp + 1);  // of a tile's queries, by warps; and of the next one's
    uint64_t* bars = reinterpret_cast<uint64_t*>(qrange + 8);
    uint32_t* slot_tmem = reinterpret_cast<uint32_t*>(bars + 2);
    volatile int* dead = reinterpret_cast<volatile int*>(slot_tmem + 1);
    const int entries = BIAS ? bias_entries(p.bias) : 0, kvh = blockIdx.y, group = p.heads / p.kv_heads, z = blockIdx.z;
    float* E = reinterpret_cast<float*>(base + L::kBytes);
    const uint32_t bar_s = tc::smem_addr(bars), bar_o = bar_s + 8, bar_end = bar_s + 24;

    const int tid = threadIdx.x, warp = tid >> 5, row = tid & (kRows - 1), j0 = (tid / kRows) * N;
    const int dim16 = (p.dim + 15) & ~15, slots = attn_slots(p.tk, p.windows, KT);
    const Loader<T, kThreads> ok(p.k, p.k_st, p.k_sh, p.dim, kvh), ov(p.v, p.v_st, p.v_sh, p.dim, kvh),
        oq(p.q, p.q_st, p.q_sh, p.dim, kvh * group), og(p.dout, p.do_st, p.do_sh, p.dim, kvh * group);
    if (tid == 0) {
        tc::mbar_init(bar_s, 1);
        tc::mbar_init(bar_o, 1);
        tc::mbar_init(bar_end, 1);
        tc::mbar_init_fence();
        *dead = 0;
    }
    if (warp == 0) tc::tmem_alloc<L::kCols>(tc::smem_addr(slot_tmem));
    tc::fence_before();
    __syncthreads();
    tc::fence_after();
    const uint32_t tmem = *slot_tmem, ts = tmem + (static_cast<uint32_t>((warp & 3) * 32) << 16);
    const uint32_t t_dv = 2 * KT, t_dk = 2 * KT + DP;
    const uint32_t id_grad = tc::idesc(kIsBf16<T>, dim16, true, true);
    int par_s = 0, par_o = 0, head_of_E = -1;
    bool alive = true;
    // dk and dv through smem where their rows are not on 16 bytes (there, direct stores were 2% faster)
    const bool staged = p.qsplits == 1 &&
                        ((p.dim & 7) != 0 || ((reinterpret_cast<uintptr_t>(p.dk) | reinterpret_cast<uintptr_t>(p.dv)) & 15) != 0);

    AttnWalk<KT> walk;
    for (bool more = walk_range(walk, slots, p, p.k_off, p.tk, p.q_off, p.tq); more; more = walk.next()) {
        const AttnTile& t = walk.tile;
        if (t.window < 0 || t.len <= p.short_max) continue;
        const float up = ds_scale<T>(p, t.window, kvh);
        const int lq = t.olen, lk = t.len, n = min(KT, lk - t.first), n16 = (n + 15) & ~15;
        const int qtiles = (lq + kRows - 1) / kRows, total = group * qtiles, per = (total + p.qsplits - 1) / p.qsplits;
        const int i0 = min(z * per, total), i1 = min(i0 + per, total);
        // causal: query tiles before this one see none of the tile's keys
        const int qt0 = p.causal ? min(max(t.first - (lk - lq), 0) / kRows, qtiles) : 0;
        auto next = [&](int it) { return it < i1 && it % qtiles < qt0 ? it - it % qtiles + qt0 : it; };
        auto fetch = [&](int it) {
            const int first = (it % qtiles) * kRows, rows = min(kRows, lq - first);
            oq.load(sq, kRows, t.obegin + first, rows, kRows, (it / qtiles) * p.q_sh);
            og.load(sg, kRows, t.obegin + first, rows, kRows, (it / qtiles) * p.do_sh);
        };
        // What a thread knows of its query of a tile; asked for a tile ahead.
        struct Row {
            float lse, delta, far;
            int2 qp;
        };
        auto row_of = [&](int it) {
            const int head = kvh * group + it / qtiles, first = (it % qtiles) * kRows, rows = min(kRows, lq - first);
            const int64_t token = t.obegin + first + min(row, rows - 1), at = static_cast<int64_t>(head) * p.tq + token;
            const float lse = p.lse[at];
            return Row{lse, p.delta[at], far_factor(p, at, lse), BIAS ? bias_pos(p.bias.q_pos, p.bias.axes, token) : make_int2(0, 0)};
        };
        auto post_range = [&](const Row& r, int half) {
            const Range x = warp_range(r.qp);
            if (tid < kRows && (tid & 31) == 0) qrange[4 * half + warp] = x;
        };
        auto load_E = [&](int it) {
            head_of_E = kvh * group + it / qtiles;
            for (int e = tid; e < entries; e += kThreads) E[e] = bias_entry(p.bias, p.heads, head_of_E, e);
        };
        // Of the queries in smem, once everyone's copies are there. False: a wait has run out, nothing more is issued.
        auto scores = [&] {
            tc::cp_async_wait<0>();
            tc::fence_async();
            tc::fence_before();
            if (__syncthreads_or(!alive)) return false;
            if (warp == 0 && tc::elect_one()) {
                tc::fence_after();
                const uint32_t id = tc::idesc(kIsBf16<T>, n16, false, false);
                tc::mma_nt<DP, kRows, KT>(tmem, sq, sk, dim16, id);
                tc::mma_nt<DP, kRows, KT>(tmem + KT, sg, sv, dim16, id);
                tc::commit(bar_s);
            }
            return true;
        };
        __syncthreads();
        int it = next(i0), half = 0;
        const bool any = it < i1;
        bool issued = false;  // the scores of `it`; the same in every thread
        Row now{};
        if (any) {
            ok.load(sk, KT, t.begin + t.first, n, n16);
            ov.load(sv, KT, t.begin + t.first, n, n16);
            fetch(it);
            tc::cp_async_commit();
            now = row_of(it);
            if (BIAS) {
                load_key_pos<KT>(kp, p.bias, t.begin + t.first, n);
                post_range(now, 0);
                if (kvh * group + it / qtiles != head_of_E) load_E(it);
            }
            issued = scores();
        }
        bool begun = false;
        while (issued && it < i1) {
            const int first = (it % qtiles) * kRows, rows = min(kRows, lq - first), after = next(it + 1);
            const bool live = row < rows;
            Row ahead{};
            if (after < i1) ahead = row_of(after);
            const int see = !live ? 0 : p.causal ? min(max(first + row + lk - lq + 1, 0), lk) : lk;
            const bool whole = n == n16 && (!p.causal || first + lk - lq + 1 >= t.first + n);
            BiasMode mode = kOne;
            if (BIAS) {
                const Range* r = qrange + 4 * half;
                mode = bias_mode(p.bias, join(join(r[0], r[1]), join(r[2], r[3])), key_range(kp));
            }
            alive = tc::mbar_wait(bar_s, par_s, dead) && alive;
            par_s ^= 1;
            tc::fence_after();
            float s[N], dp[N];
            weights<KT, BIAS>(p, s, dp, ts, ts + KT, n16, j0, whole, see - t.first, live ? now.lse : INFINITY, now.far, mode, E, kp, now.qp);
            write_row<T>(sp, row, j0, s, 1.0f);
            score_gradients(s, dp, live ? now.delta : 0.0f, j0, whole, see - t.first);
            write_row<T>(sd, row, j0, dp, up);
            if (BIAS && after < i1) post_range(ahead, half ^ 1);
            tc::fence_async();
            tc::fence_before();
            __syncthreads();
            if (warp == 0 && tc::elect_one()) {
                tc::fence_after();
                tc::mma_tt<kRows>(tmem + t_dv, tc::desc(sp, kRows * 128), tc::desc(sg, kRows * 128), id_grad, begun);
                tc::mma_tt<kRows>(tmem + t_dk, tc::desc(sd, kRows * 128), tc::desc(sq, kRows * 128), id_grad, begun);
                tc::commit(bar_o);
            }
            if (BIAS && after < i1 && kvh * group + after / qtiles != head_of_E) load_E(after);  // everyone is past this head's lookups
            alive = tc::mbar_wait(bar_o, par_o, dead) && alive;
            par_o ^= 1;
            begun = true;
            if (after < i1) {
                fetch(after);
                tc::cp_async_commit();
                issued = scores();
            }
            it = after, now = ahead, half ^= 1;
        }
        tc::fence_after();
        if (__syncthreads_or(!alive)) alive = false;  // one thread's weights are in every row
        const bool of_v = tid < kRows;
        const int64_t key = t.begin + t.first + min(row, n - 1);
        const bool odd = tid < 2 * kRows && finish_key_row<T, DP>(p, ts + (of_v ? t_dv : t_dk), row < n, any, key, kvh, z, up,
                                                                   of_v, alive, staged, of_v ? sp : sd, row);
        if (staged) {
            __syncthreads();
            store_panel<T, kThreads>(sp, p.dv, p.kv_heads, p.dim, t.begin, kvh, 1, t.first, n);
            store_panel<T, kThreads>(sd, p.dk, p.kv_heads, p.dim, t.begin, kvh, 1, t.first, n);
            if (p.causal) __syncthreads();  // before rows that are written once more
        }
        if (p.causal && tid < 2 * kRows && key_again<T>(p, odd, t.first + row, kvh, t.obegin, lq, lk, qt0, i0, i1, of_v))
            key_row<T>(p, key, t.first + row, kvh, t.obegin, lq, lk, i0, i1, up, of_v, z);
        tc::fence_before();
    }
    const bool lost = __syncthreads_or(!alive);
    tc::fence_before();
    finish_block(lost, bar_end);
    if (warp == 0) tc::tmem_free<L::kCols>(tmem);
}

// ---- sums across blocks ------------------------------------------------------------------------
template <typename T>
__global__ void __launch_bounds__(256) k_attn_join_dkv(AttnParams p) {
    const int64_t n = static_cast<int64_t>(p.tk) * p.kv_heads * p.dim;
    const int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
    if (i >= n) return;
    float k = 0.0f, v = 0.0f;
    for (int s = 0; s < p.qsplits; ++s) {
        k += p.part_dk[s * n + i];
        v += p.part_dv[s * n + i];
    }
    static_cast<T*>(p.dk)[i] = from_f<T>(k);
    static_cast<T*>(p.dv)[i] = from_f<T>(v);
}

template <typename T, int DP, bool BIAS>
cudaError_t bwd_one(const AttnParams& p, void* dtable, cudaStream_t s) {
    const int entries = bias_entries(p.bias), group = p.heads / p.kv_heads, sum = p.bias_part != nullptr;
    cudaError_t err;
    const int b_short = 1024 + ShortSmem<DP>::kBytes + entries * group * (4 + 8 * sum) + entries * 4 * sum;
    if (p.tiny_blocks > 0 && (err = launch_attn_backward_tiny(p, std::is_same<T, __half>::value ? kF16 : kBF16, s)) != cudaSuccess) return err;
    if (p.short_max == 0) {
        // only rows and windows without partners: no bias is looked up
        const int bytes = 1024 + ShortSmem<DP>::kBytes;
        if ((err = allow_smem(k_attn_bwd_short<T, DP, false>)) != cudaSuccess) return err;
        k_attn_bwd_short<T, DP, false><<<dim3(p.short_blocks, p.kv_heads, 1), 2 * kRows, bytes, s>>>(p);
    } else {
        if ((err = allow_smem(k_attn_bwd_short<T, DP, BIAS>)) != cudaSuccess) return err;
        k_attn_bwd_short<T, DP, BIAS><<<dim3(p.short_blocks, p.kv_heads, p.qsplits), 2 * kRows, b_short, s>>>(p);
    }
    if ((err = cudaGetLastError()) != cudaSuccess) return err;
    const int b_dq = 1024 + DqShape<DP>::kBytes + entries * (4 + 12 * sum);
    if ((err = allow_smem(k_attn_dq_long<T, DP, BIAS>)) != cudaSuccess) return err;
    k_attn_dq_long<T, DP, BIAS><<<dim3(p.dq_blocks, p.heads), DqShape<DP>::kThreads, b_dq, s>>>(p);
    if ((err = cudaGetLastError()) != cudaSuccess) return err;
    const int b_kv = 1024 + DkvShape<DP>::kBytes + entries * 4;
    if ((err = allow_smem(k_attn_dkv_long<T, DP, BIAS>)) != cudaSuccess) return err;
    k_attn_dkv_long<T, DP, BIAS><<<dim3(p.dkv_blocks, p.kv_heads, p.qsplits), DkvShape<DP>::kThreads, b_kv, s>>>(p);
    if ((err = cudaGetLastError()) != cudaSuccess) return err;
    if (p.qsplits > 1) {
        const int64_t n = static_cast<int64_t>(p.tk) * p.kv_heads * p.dim;
        k_attn_join_dkv<T><<<static_cast<unsigned>((n + 255) / 256), 256, 0, s>>>(p);
        if ((err = cudaGetLastError()) != cudaSuccess) return err;
    }
    return dtable != nullptr ? launch_attn_bias_grad(p, dtable, s) : cudaSuccess;
}

template <typename T>
cudaError_t bwd_type(const AttnParams& p, void* dtable, cudaStream_t s) {
    if (p.bias.table != nullptr) return p.dim <= 64 ? bwd_one<T, 64, true>(p, dtable, s) : bwd_one<T, 128, true>(p, dtable, s);
    return p.dim <= 64 ? bwd_one<T, 64, false>(p, dtable, s) : bwd_one<T, 128, false>(p, dtable, s);
}

}  // namespace

cudaError_t launch_attn_backward_mma(const AttnParams& p, int type, void* dtable, int sms, cudaStream_t s) {
    if (p.tiny_max > 0)
        k_attn_lists<<<1, 1024, 0, s>>>(p, p.flags);
    else
        k_attn_flags<<<p.windows < 16384 ? 1 + p.windows / 1024 : 16, 256, 0, s>>>(p, p.flags);
    cudaError_t err = cudaGetLastError();
    if (err != cudaSuccess) return err;
    if (p.win_max != nullptr) {
        const int q_slots = attn_slots(p.tq, p.windows, kRows), k_slots = attn_slots(p.tk, p.windows, kRows);
        k_attn_window_max<<<q_slots + k_slots, 256, 0, s>>>(p, q_slots);
        if ((err = cudaGetLastError()) != cudaSuccess) return err;
    }
    if ((err = launch_attn_delta(p, type, sms, s)) != cudaSuccess) return err;
    return type == kBF16 ? bwd_type<__nv_bfloat16>(p, dtable, s) : bwd_type<__half>(p, dtable, s);
}

cudaError_t attn_timeouts_bwd(unsigned int* count) {
    return cudaMemcpyFromSymbol(count, g_timeouts, sizeof(unsigned int));
}

}  // namespace oss
