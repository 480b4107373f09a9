// The norms before and after a block, fused with its gate and residual scale:
//   n = norm(h) w + b,   y = x + s a(gate) n,   z = norm(y) w' + b'
// and the backward of the three. norm(u) = (u - mean) r (layer) or u r (rms).
//
// Each row belongs to a group of lanes (8, 16 or 32 of a warp, or a whole block for rows of
// more than 256 channels, of up to 256 threads or 1024); a lane keeps its 8 columns of the row and
// of the parameters in registers, so that a call reads every activation once and writes every
// result once. Blocks stay and walk rows; the next row's values are on their way
// while one is worked on. The backward takes x, h and the gate again and recomputes n and y in
// fp32 (y as written would carry its rounding into every gradient), with the means and deviations
// of the forward. Sums over rows go lane by lane in fp32 (one lane adds at most rows / groups terms),
// over the groups of a block in order, then over the blocks in double, always in the same order.
// 522240 rows of 128 in bf16 with a full gate, forward: 148 us, 4.5 TB/s, 69% of a copy's (271 us without the next
// row's values on their way); the latency of its loads bounds it, at 37% of an SM's warps. 32640 rows of 1024 in bf16,
// silu gate, forward and backward: 353 us, 1.9 TB/s; the backward's 128 registers leave 24% of the warps, too few for
// its loads.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "internal.h"
#include "gated_norm.cuh"

namespace oss {
namespace {

constexpr int kElems = 8;     // columns of a lane
constexpr int kGroup = 256;   // threads of a block that holds several rows

template <typename T, int V>
struct alignas(sizeof(T) * V) Pack {
    T v[V];
};

__device__ __forceinline__ float up(float x) { return x; }
__device__ __forceinline__ float up(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float up(__half x) { return __half2float(x); }
__device__ __forceinline__ void down(float& y, float x) { y = x; }
__device__ __forceinline__ void down(__nv_bfloat16& y, float x) { y = __float2bfloat16_rn(x); }
__device__ __forceinline__ void down(__half& y, float x) { y = __float2half_rn(x); }

// Column of element i of a lane: vectors of V, a group's lanes side by side.
template <int V>
__device__ __forceinline__ int col_of(int lane, int lanes, int i) {
    return ((i / V) * lanes + lane) * V + (i % V);
}

// A row's values as loaded. FULL: the lanes' columns end with the row.
template <typename T, int V>
struct Raw {
    Pack<T, V> v[kElems / V];
};
template <typename T, int V, bool FULL>
__device__ __forceinline__ void fetch_row(Raw<T, V>& r, const T* p, bool live, int lane, int lanes, int c) {
#pragma unroll
    for (int i = 0; i < kElems; i += V) {
        const int col = col_of<V>(lane, lanes, i);
        if (live && (FULL || col < c)) r.v[i / V] = *reinterpret_cast<const Pack<T, V>*>(p + col);
    }
}
template <typename T, int V, bool FULL>
__device__ __forceinline__ void unpack_row(float (&out)[kElems], const Raw<T, V>& r, bool live, int lane, int lanes, int c) {
#pragma unroll
    for (int i = 0; i < kElems; i += V) {
        const bool on = live && (FULL || col_of<V>(lane, lanes, i) < c);
#pragma unroll
        for (int v = 0; v < V; ++v) out[i + v] = on ? up(r.v[i / V].v[v]) : 0.0f;
    }
}
template <typename T, int V, bool FULL>
__device__ __forceinline__ void store_row(T* p, const float (&in)[kElems], bool live, int lane, int lanes, int c) {
#pragma unroll
    for (int i = 0; i < kElems; i += V) {
        const int col = col_of<V>(lane, lanes, i);
        if (live && (FULL || col < c)) {
            Pack<T, V> t;
#pragma unroll
            for (int v = 0; v < V; ++v) down(t.v[v], in[i + v]);
            *reinterpret_cast<Pack<T, V>*>(p + col) = t;
        }
    }
}

// Parameters are read once a block, an element at a time.
template <int V>
__device__ __forceinline__ void load_param(float (&out)[kElems], const void* p, int type, float absent, int lane, int lanes, int c) {
#pragma unroll
    for (int i = 0; i < kElems; ++i) {
        const int col = col_of<V>(lane, lanes, i);
        float x = absent;
        if (p != nullptr && col < c)
            x = type == 0   ? static_cast<const float*>(p)[col]
                : type == 1 ? __bfloat162float(static_cast<const __nv_bfloat16*>(p)[col])
                            : __half2float(static_cast<const __half*>(p)[col]);
        out[i] = col < c ? x : 0.0f;
    }
}

// Sums of K values over the lanes of a row, the same in each of them. `turn` alternates between the
// two halves of `shared` (of 32 K_MAX floats each), so that one barrier a sum is enough.
constexpr int kMostSums = 3;
template <int TPR, int K>
__device__ __forceinline__ void row_sum(float (&v)[K], float* shared, int& turn) {
    constexpr int W = TPR <= 0 ? 32 : TPR;
#pragma unroll
    for (int x = W / 2; x > 0; x >>= 1)
#pragma unroll
        for (int k = 0; k < K; ++k) v[k] += __shfl_xor_sync(0xffffffffu, v[k], x);
    if constexpr (TPR <= 0) {  // the whole block
        const int warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
        float* at = shared + turn * 32 * kMostSums;
        turn ^= 1;
        if ((threadIdx.x & 31) == 0)
#pragma unroll
            for (int k = 0; k < K; ++k) at[k * 32 + warp] = v[k];
        __syncthreads();
#pragma unroll
        for (int k = 0; k < K; ++k) {
            float s = 0.0f;
            for (int w = 0; w < warps; ++w) s += at[k * 32 + w];
            v[k] = s;
        }
    }
}

// mean and 1 / deviation of a row; the deviation from centred values (a lane's absent columns
// are left out).
template <int TPR, int V, bool FULL, bool LAYER>
__device__ __forceinline__ float2 row_stats(const float (&u)[kElems], const GatedNorm& p, int lane, int lanes, float* shared, int& turn) {
    float mean = 0.0f;
    if (LAYER) {
        float s[1] = {0.0f};
#pragma unroll
        for (int i = 0; i < kElems; ++i) s[0] += u[i];
        row_sum<TPR>(s, shared, turn);
        mean = s[0] * p.inv_c;
    }
    float q[1] = {0.0f};
#pragma unroll
    for (int i = 0; i < kElems; ++i) {
        const float d = !LAYER ? u[i] : FULL || col_of<V>(lane, lanes, i) < p.c ? u[i] - mean : 0.0f;
        q[0] = fmaf(d, d, q[0]);
    }
    row_sum<TPR>(q, shared, turn);
    return make_float2(mean, rsqrtf(q[0] * p.inv_c + p.eps));
}

// The gate's values to their activations, and with SLOPE to its slopes as well. For 16-bit values __expf, off by 2^-21 and
// more the farther from 0, and a quotient that is 0 beyond 2^126 are far below a rounding of theirs; fp32 values
// get expf of a negative number, right to their last digits at either end.
template <bool SLOPE, bool EXACT>
__device__ __forceinline__ void activate(float (&g)[kElems], float (&slope)[kElems], int act) {
    if (act == 0) {
#pragma unroll
        for (int i = 0; i < kElems; ++i) slope[i] = 1.0f;
        return;
    }
#pragma unroll
    for (int i = 0; i < kElems; ++i) {
        float s;
        if (EXACT) {
            const float t = expf(-fabsf(g[i]));
            s = (g[i] < 0.0f ? t : 1.0f) / (1.0f + t);
        } else {
            s = __fdividef(1.0f, 1.0f + __expf(-g[i]));
        }
        if (act == 1) {
            if (SLOPE) slope[i] = s * (1.0f - s);
            g[i] = s;
        } else {
            if (SLOPE) slope[i] = s * (1.0f + g[i] * (1.0f - s));
            g[i] *= s;
        }
    }
}

template <typename T, int TPR, int V, bool FULL, bool LAYER>
__global__ void __launch_bounds__(TPR < 0 ? 1024 : kGroup, TPR < 0 ? 1 : 3) k_gated_norm_fwd(GatedNorm p) {
    __shared__ float shared[TPR <= 0 ? 2 * 32 * kMostSums : 1];
    const int lanes = TPR <= 0 ? static_cast<int>(blockDim.x) : TPR, groups = static_cast<int>(blockDim.x) / lanes;
    const int lane = threadIdx.x % lanes, group = threadIdx.x / lanes;
    int turn = 0;
    float w[kElems], b[kElems] = {}, s[kElems], w2[kElems], b2[kElems] = {};
    load_param<V>(w, p.weight, p.param_type, 1.0f, lane, lanes, p.c);
    if (LAYER) load_param<V>(b, p.bias, p.param_type, 0.0f, lane, lanes, p.c);
    load_param<V>(s, p.scale, p.param_type, 1.0f, lane, lanes, p.c);
    load_param<V>(w2, p.next_weight, p.param_type, 1.0f, lane, lanes, p.c);
    if (LAYER) load_param<V>(b2, p.next_bias, p.param_type, 0.0f, lane, lanes, p.c);
#pragma unroll
    for (int i = 0; i < kElems; ++i) {  // scale (n w + b), the gate to come
        w[i] *= s[i];
        if (LAYER) b[i] *= s[i];
    }
    Raw<T, V> rx, rh, rg;
    float one = 1.0f;
    auto fetch = [&](int64_t row) {
        const bool on = row < p.rows;
        fetch_row<T, V, FULL>(rh, static_cast<const T*>(p.h) + row * p.h_st, on, lane, lanes, p.c);
        fetch_row<T, V, FULL>(rx, static_cast<const T*>(p.x) + row * p.x_st, on, lane, lanes, p.c);
        if (p.gate_kind == 2) fetch_row<T, V, FULL>(rg, static_cast<const T*>(p.gate) + row * p.g_st, on, lane, lanes, p.c);
        if (p.gate_kind == 1) one = on ? up(static_cast<const T*>(p.gate)[row * p.g_st]) : 1.0f;
    };
    const int64_t step = static_cast<int64_t>(gridDim.x) * groups;
    int64_t row = static_cast<int64_t>(blockIdx.x) * groups + group;
    fetch(row);
    // whole blocks stay in the loop: the shuffles name every lane
    for (int64_t row0 = static_cast<int64_t>(blockIdx.x) * groups; row0 < p.rows; row0 += step, row += step) {
        const bool live = row < p.rows;
        float x[kElems], h[kElems], g[kElems], slope[kElems];
        unpack_row<T, V, FULL>(h, rh, live, lane, lanes, p.c);
        unpack_row<T, V, FULL>(x, rx, live, lane, lanes, p.c);
        if (p.gate_kind == 2) {
            unpack_row<T, V, FULL>(g, rg, live, lane, lanes, p.c);
        } else {
#pragma unroll
            for (int i = 0; i < kElems; ++i) g[i] = one;
        }
        fetch(row + step);
        activate<false, sizeof(T) == 4>(g, slope, p.act);
        const float2 st1 = row_stats<TPR, V, FULL, LAYER>(h, p, lane, lanes, shared, turn);
#pragma unroll
        for (int i = 0; i < kElems; ++i) x[i] = fmaf(g[i], LAYER ? fmaf((h[i] - st1.x) * st1.y, w[i], b[i]) : h[i] * st1.y * w[i], x[i]);
        store_row<T, V, FULL>(static_cast<T*>(p.y) + row * p.c, x, live, lane, lanes, p.c);
        float2 st2 = make_float2(0.0f, 0.0f);
        if (p.z != nullptr) {
            st2 = row_stats<TPR, V, FULL, LAYER>(x, p, lane, lanes, shared, turn);
#pragma unroll
            for (int i = 0; i < kElems; ++i) x[i] = LAYER ? fmaf((x[i] - st2.x) * st2.y, w2[i], b2[i]) : x[i] * st2.y * w2[i];
            store_row<T, V, FULL>(static_cast<T*>(p.z) + row * p.c, x, live, lane, lanes, p.c);
        }
        if (p.stats != nullptr && live && lane == 0) p.stats[row] = make_float4(st1.x, st1.y, st2.x, st2.y);
    }
}

template <typename T, int TPR, int V, bool FULL, bool LAYER>
__global__ void __launch_bounds__(TPR < 0 ? 1024 : kGroup, TPR < 0 ? 1 : 2) k_gated_norm_bwd(GatedNorm p) {
    __shared__ float shared[TPR <= 0 ? 2 * 32 * kMostSums : kGroup * kElems];
    const int lanes = TPR <= 0 ? static_cast<int>(blockDim.x) : TPR, groups = static_cast<int>(blockDim.x) / lanes;
    const int lane = threadIdx.x % lanes, group = threadIdx.x / lanes;
    int turn = 0;
    float w[kElems], b[kElems] = {}, s[kElems], w2[kElems];
    load_param<V>(w, p.weight, p.param_type, 1.0f, lane, lanes, p.c);
    if (LAYER) load_param<V>(b, p.bias, p.param_type, 0.0f, lane, lanes, p.c);
    load_param<V>(s, p.scale, p.param_type, 1.0f, lane, lanes, p.c);
    load_param<V>(w2, p.next_weight, p.param_type, 1.0f, lane, lanes, p.c);
    float dw[kElems] = {}, db[kElems] = {}, ds[kElems] = {}, dw2[kElems] = {}, db2[kElems] = {};
    Raw<T, V> rx, rh, rg, ry, rz;
    float one = 1.0f;
    float4 rst;
    auto fetch = [&](int64_t row) {
        const bool on = row < p.rows;
        fetch_row<T, V, FULL>(rh, static_cast<const T*>(p.h) + row * p.h_st, on, lane, lanes, p.c);
        fetch_row<T, V, FULL>(rx, static_cast<const T*>(p.x) + row * p.x_st, on, lane, lanes, p.c);
        if (p.gate_kind == 2) fetch_row<T, V, FULL>(rg, static_cast<const T*>(p.gate) + row * p.g_st, on, lane, lanes, p.c);
        if (p.gate_kind == 1) one = on ? up(static_cast<const T*>(p.gate)[row * p.g_st]) : 1.0f;
        if (p.dz != nullptr) fetch_row<T, V, FULL>(rz, static_cast<const T*>(p.dz) + row * p.dz_st, on, lane, lanes, p.c);
        if (p.dy != nullptr) fetch_row<T, V, FULL>(ry, static_cast<const T*>(p.dy) + row * p.dy_st, on, lane, lanes, p.c);
        rst = on ? p.stats[row] : make_float4(0.f, 0.f, 0.f, 0.f);
    };
    const int64_t step = static_cast<int64_t>(gridDim.x) * groups;
    int64_t row = static_cast<int64_t>(blockIdx.x) * groups + group;
    fetch(row);
    for (int64_t row0 = static_cast<int64_t>(blockIdx.x) * groups; row0 < p.rows; row0 += step, row += step) {
        const bool live = row < p.rows;
        float n[kElems], y[kElems], g[kElems], d[kElems], slope[kElems];
        const float4 st = rst;
        unpack_row<T, V, FULL>(n, rh, live, lane, lanes, p.c);
        unpack_row<T, V, FULL>(y, rx, live, lane, lanes, p.c);
        if (p.gate_kind == 2) {
            unpack_row<T, V, FULL>(g, rg, live, lane, lanes, p.c);
        } else {
#pragma unroll
            for (int i = 0; i < kElems; ++i) g[i] = one;
        }
        if (p.dy != nullptr) {
            unpack_row<T, V, FULL>(d, ry, live, lane, lanes, p.c);
        } else {
#pragma unroll
            for (int i = 0; i < kElems; ++i) d[i] = 0.0f;
        }
        float u[kElems];
        if (p.dz != nullptr) unpack_row<T, V, FULL>(u, rz, live, lane, lanes, p.c);
        fetch(row + step);
        activate<true, sizeof(T) == 4>(g, slope, p.act);
        // y again, then its norm, from the forward's statistics
#pragma unroll
        for (int i = 0; i < kElems; ++i) {
            n[i] = (LAYER ? n[i] - st.x : n[i]) * st.y;
            y[i] = fmaf(g[i] * s[i], LAYER ? fmaf(n[i], w[i], b[i]) : n[i] * w[i], y[i]);
        }
        if (p.dz != nullptr) {
            float m[2] = {0.0f, 0.0f};
#pragma unroll
            for (int i = 0; i < kElems; ++i) {
                y[i] = (LAYER ? y[i] - st.z : y[i]) * st.w;  // absent columns: u is 0
                dw2[i] = fmaf(u[i], y[i], dw2[i]);
                if (LAYER) db2[i] += u[i];
                u[i] *= w2[i];
                m[0] = fmaf(u[i], y[i], m[0]);
                if (LAYER) m[1] += u[i];
            }
            row_sum<TPR>(m, shared, turn);
            m[0] *= p.inv_c;
            m[1] *= p.inv_c;
#pragma unroll
            for (int i = 0; i < kElems; ++i) d[i] = fmaf(LAYER ? u[i] - y[i] * m[0] - m[1] : u[i] - y[i] * m[0], st.w, d[i]);
        }
        if (p.dx != nullptr) store_row<T, V, FULL>(static_cast<T*>(p.dx) + row * p.c, d, live, lane, lanes, p.c);
        float m[3] = {0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int i = 0; i < kElems; ++i) {
            if (!live || (!FULL && col_of<V>(lane, lanes, i) >= p.c)) d[i] = 0.0f;
            const float t = LAYER ? fmaf(n[i], w[i], b[i]) : n[i] * w[i], e = d[i] * g[i];
            const float da = d[i] * slope[i] * (s[i] * t);
            ds[i] = fmaf(e, t, ds[i]);
            d[i] = e * s[i];  // dn
            dw[i] = fmaf(d[i], n[i], dw[i]);
            if (LAYER) db[i] += d[i];
            d[i] *= w[i];
            m[0] = fmaf(d[i], n[i], m[0]);
            if (LAYER) m[1] += d[i];
            m[2] += da;
            g[i] = da;
        }
        row_sum<TPR>(m, shared, turn);
        if (p.dgate != nullptr) {
            if (p.gate_kind == 2)
                store_row<T, V, FULL>(static_cast<T*>(p.dgate) + row * p.c, g, live, lane, lanes, p.c);
            else if (live && lane == 0)
                down(static_cast<T*>(p.dgate)[row], m[2]);
        }
        if (p.dh != nullptr) {
            m[0] *= p.inv_c;
            m[1] *= p.inv_c;
#pragma unroll
            for (int i = 0; i < kElems; ++i) d[i] = (LAYER ? d[i] - n[i] * m[0] - m[1] : d[i] - n[i] * m[0]) * st.y;
            store_row<T, V, FULL>(static_cast<T*>(p.dh) + row * p.c, d, live, lane, lanes, p.c);
        }
    }
    // a row of partial sums for each block: [5][gridDim.x][c]
    auto finish = [&](const float (&sum)[kElems], int which) {
        float* to = p.partial + (static_cast<int64_t>(which) * gridDim.x + blockIdx.x) * p.c;
        if constexpr (TPR <= 0) {
#pragma unroll
            for (int i = 0; i < kElems; ++i) {
                const int col = col_of<V>(lane, lanes, i);
                if (col < p.c) to[col] = sum[i];
            }
        } else {
            __syncthreads();
#pragma unroll
            for (int i = 0; i < kElems; ++i) shared[group * lanes * kElems + col_of<V>(lane, lanes, i)] = sum[i];
            __syncthreads();
            for (int col = threadIdx.x; col < p.c; col += kGroup) {
                float total = 0.0f;
                for (int k = 0; k < groups; ++k) total += shared[k * lanes * kElems + col];
                to[col] = total;
            }
        }
    };
    finish(dw, 0);
    finish(ds, 1);
    finish(dw2, 2);
    if (LAYER) {
        finish(db, 3);
        finish(db2, 4);
    }
}

// Columns of the partial sums, 32 at a time: warp k adds the rows k, k + 32, ... in double,
// then the 32 sums are added in order.
__global__ void __launch_bounds__(1024) k_gated_norm_reduce(GatedNorm p, int64_t parts) {
    __shared__ double sums[32][33];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, col = blockIdx.x * 32 + lane;
    void* out = p.dparam[blockIdx.y];
    if (out == nullptr) return;
    double sum = 0.0;
    if (col < p.c) {
        const float* at = p.partial + static_cast<int64_t>(blockIdx.y) * parts * p.c + col;
        #pragma unroll 4
        for (int64_t r = warp; r < parts; r += 32) sum += static_cast<double>(at[r * p.c]);
    }
    sums[warp][lane] = sum;
    __syncthreads();
    if (warp != 0 || col >= p.c) return;
    for (int w = 1; w < 32; ++w) sum += sums[w][lane];
    if (p.param_type == 0)
        static_cast<float*>(out)[col] = static_cast<float>(sum);
    else if (p.param_type == 1)
        static_cast<__nv_bfloat16*>(out)[col] = __double2bfloat16(sum);
    else
        static_cast<__half*>(out)[col] = __double2half(sum);
}

struct Shape {
    int tpr;      // lanes of a row, 0: a block of up to 256, -1: of up to 1024
    int threads;  // of a block
    int groups;   // rows that a block holds at once
    int64_t blocks;
};
Shape shape_of(int64_t rows, int c, int most) {
    Shape s;
    const int lanes = (c + kElems - 1) / kElems;
    s.tpr = lanes <= 8 ? 8 : lanes <= 16 ? 16 : lanes <= 32 ? 32 : lanes <= kGroup ? 0 : -1;
    s.threads = s.tpr > 0 ? kGroup : (lanes + 31) / 32 * 32;
    s.groups = s.tpr > 0 ? kGroup / s.tpr : 1;
    // as many blocks as stay resident with `most` threads on each of the 148 SMs
    const int64_t resident = 148ll * (most / s.threads < 1 ? 1 : most / s.threads);
    const int64_t want = (rows + s.groups - 1) / s.groups;
    s.blocks = want < resident ? want : resident;
    return s;
}
constexpr int kFwdThreads = 3 * kGroup, kBwdThreads = 2 * kGroup;

template <typename T, int V, bool FULL, bool LAYER>
void fwd_full(const GatedNorm& p, const Shape& sh, cudaStream_t s) {
    const unsigned g = static_cast<unsigned>(sh.blocks);
    if (sh.tpr == 8)
        k_gated_norm_fwd<T, 8, V, FULL, LAYER><<<g, sh.threads, 0, s>>>(p);
    else if (sh.tpr == 16)
        k_gated_norm_fwd<T, 16, V, FULL, LAYER><<<g, sh.threads, 0, s>>>(p);
    else if (sh.tpr == 32)
        k_gated_norm_fwd<T, 32, V, FULL, LAYER><<<g, sh.threads, 0, s>>>(p);
    else if (sh.tpr == 0)
        k_gated_norm_fwd<T, 0, V, FULL, LAYER><<<g, sh.threads, 0, s>>>(p);
    else
        k_gated_norm_fwd<T, -1, V, FULL, LAYER><<<g, sh.threads, 0, s>>>(p);
}
template <typename T, int V>
cudaError_t fwd_vec(const GatedNorm& p, cudaStream_t s) {
    const Shape sh = shape_of(p.rows, p.c, kFwdThreads);
    if (V > 1 && (sh.tpr > 0 ? sh.tpr : sh.threads) * kElems == p.c)
        p.layer ? fwd_full<T, V, V != 1, true>(p, sh, s) : fwd_full<T, V, V != 1, false>(p, sh, s);
    else
        p.layer ? fwd_full<T, V, false, true>(p, sh, s) : fwd_full<T, V, false, false>(p, sh, s);
    return cudaGetLastError();
}
template <typename T, int V, bool FULL, bool LAYER>
void bwd_full(const GatedNorm& p, const Shape& sh, cudaStream_t s) {
    const unsigned g = static_cast<unsigned>(sh.blocks);
    if (sh.tpr == 8)
        k_gated_norm_bwd<T, 8, V, FULL, LAYER><<<g, sh.threads, 0, s>>>(p);
    else if (sh.tpr == 16)
        k_gated_norm_bwd<T, 16, V, FULL, LAYER><<<g, sh.threads, 0, s>>>(p);
    else if (sh.tpr == 32)
        k_gated_norm_bwd<T, 32, V, FULL, LAYER><<<g, sh.threads, 0, s>>>(p);
    else if (sh.tpr == 0)
        k_gated_norm_bwd<T, 0, V, FULL, LAYER><<<g, sh.threads, 0, s>>>(p);
    else
        k_gated_norm_bwd<T, -1, V, FULL, LAYER><<<g, sh.threads, 0, s>>>(p);
}
template <typename T, int V>
cudaError_t bwd_vec(const GatedNorm& p, cudaStream_t s) {
    const Shape sh = shape_of(p.rows, p.c, kBwdThreads);
    if (V > 1 && (sh.tpr > 0 ? sh.tpr : sh.threads) * kElems == p.c)
        p.layer ? bwd_full<T, V, V != 1, true>(p, sh, s) : bwd_full<T, V, V != 1, false>(p, sh, s);
    else
        p.layer ? bwd_full<T, V, false, true>(p, sh, s) : bwd_full<T, V, false, false>(p, sh, s);
    cudaError_t err = cudaGetLastError();
    if (err != cudaSuccess) return err;
    k_gated_norm_reduce<<<dim3((p.c + 31) / 32, p.layer ? 5 : 3), 1024, 0, s>>>(p, sh.blocks);
    return cudaGetLastError();
}

// 16-byte vectors where every row of every operand starts on one.
bool vectors(const GatedNorm& p, int elem) {
    const int v = 16 / elem;
    const void* ptrs[] = {p.x, p.h, p.gate_kind == 2 ? p.gate : nullptr, p.dy, p.dz, p.y, p.z, p.dx, p.dh,
                          p.gate_kind == 2 ? p.dgate : nullptr};
    for (const void* q : ptrs)
        if (reinterpret_cast<uintptr_t>(q) & 15) return false;
    return p.c % v == 0 && p.x_st % v == 0 && p.h_st % v == 0 && (p.gate_kind != 2 || p.g_st % v == 0) && p.dy_st % v == 0 &&
           p.dz_st % v == 0;
}

}  // namespace

int64_t gated_norm_partial_floats(int64_t rows, int c) {
    const Shape s = shape_of(rows, c, kBwdThreads);
    return 5 * s.blocks * c;
}

cudaError_t launch_gated_norm_forward(const GatedNorm& p, int type, cudaStream_t s) {
    const bool v = vectors(p, type == 0 ? 4 : 2);
    if (type == 0) return v ? fwd_vec<float, 4>(p, s) : fwd_vec<float, 1>(p, s);
    if (type == 1) return v ? fwd_vec<__nv_bfloat16, 8>(p, s) : fwd_vec<__nv_bfloat16, 1>(p, s);
    return v ? fwd_vec<__half, 8>(p, s) : fwd_vec<__half, 1>(p, s);
}

cudaError_t launch_gated_norm_backward(const GatedNorm& p, int type, cudaStream_t s) {
    const bool v = vectors(p, type == 0 ? 4 : 2);
    if (type == 0) return v ? bwd_vec<float, 4>(p, s) : bwd_vec<float, 1>(p, s);
    if (type == 1) return v ? bwd_vec<__nv_bfloat16, 8>(p, s) : bwd_vec<__nv_bfloat16, 1>(p, s);
    return v ? bwd_vec<__half, 8>(p, s) : bwd_vec<__half, 1>(p, s);
}

}  // namespace oss
