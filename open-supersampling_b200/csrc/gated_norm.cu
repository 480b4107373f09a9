// The norms before and after a block, fused with its gate and residual scale:
//   n = norm(h) w + b,   y = x + s a(gate) n,   z = norm(y) w' + b'
// and the backward of the three. norm(u) = (u - mean) r (layer) or u r (rms).
//
// Each row belongs to a group of lanes (8, 16 or 32 of a warp, or a whole block for rows of
// more than 256 channels, of up to 256 threads or 1024); a lane keeps its 8 columns of the row and of the parameters in
// registers, so that a call reads every activation once and writes every result once: HBM
// bounds it. The backward takes x, h and the gate again and recomputes n and y in fp32 (y as
// written would carry its rounding into every gradient), with the means and deviations of the
// forward. Sums over rows go lane by lane in fp32 (one lane adds at most rows / groups terms),
// then over the groups in double, always in the same order.
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

template <typename T, int V>
__device__ __forceinline__ void load_row(float (&out)[kElems], const T* p, int lane, int lanes, int c) {
#pragma unroll
    for (int i = 0; i < kElems; i += V) {
        const int col = col_of<V>(lane, lanes, i);
        if (col < c) {
            const Pack<T, V> t = *reinterpret_cast<const Pack<T, V>*>(p + col);
#pragma unroll
            for (int v = 0; v < V; ++v) out[i + v] = up(t.v[v]);
        } else {
#pragma unroll
            for (int v = 0; v < V; ++v) out[i + v] = 0.0f;
        }
    }
}
template <typename T, int V>
__device__ __forceinline__ void store_row(T* p, const float (&in)[kElems], int lane, int lanes, int c) {
#pragma unroll
    for (int i = 0; i < kElems; i += V) {
        const int col = col_of<V>(lane, lanes, i);
        if (col < c) {
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

// Sums of K values over the lanes of a row, the same in each of them.
template <int TPR, int K>
__device__ __forceinline__ void row_sum(float (&v)[K], float* shared) {
    constexpr int W = TPR <= 0 ? 32 : TPR;
#pragma unroll
    for (int x = W / 2; x > 0; x >>= 1)
#pragma unroll
        for (int k = 0; k < K; ++k) v[k] += __shfl_xor_sync(0xffffffffu, v[k], x);
    if constexpr (TPR <= 0) {  // the whole block
        const int warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
        __syncthreads();
        if ((threadIdx.x & 31) == 0)
#pragma unroll
            for (int k = 0; k < K; ++k) shared[k * 32 + warp] = v[k];
        __syncthreads();
#pragma unroll
        for (int k = 0; k < K; ++k) {
            float s = 0.0f;
            for (int w = 0; w < warps; ++w) s += shared[k * 32 + w];
            v[k] = s;
        }
    }
}

// mean and 1 / deviation of a row; the deviation from centred values (a lane's absent columns
// are left out).
template <int TPR, int V>
__device__ __forceinline__ float2 row_stats(const float (&u)[kElems], const GatedNorm& p, int lane, int lanes, float* shared) {
    float mean = 0.0f;
    if (p.layer) {
        float s[1] = {0.0f};
#pragma unroll
        for (int i = 0; i < kElems; ++i) s[0] += u[i];
        row_sum<TPR>(s, shared);
        mean = s[0] * p.inv_c;
    }
    float q[1] = {0.0f};
#pragma unroll
    for (int i = 0; i < kElems; ++i) {
        const float d = col_of<V>(lane, lanes, i) < p.c ? u[i] - mean : 0.0f;
        q[0] = fmaf(d, d, q[0]);
    }
    row_sum<TPR>(q, shared);
    return make_float2(mean, rsqrtf(q[0] * p.inv_c + p.eps));
}

__device__ __forceinline__ float gate_value(float g, int act, float& slope) {
    if (act == 0) {
        slope = 1.0f;
        return g;
    }
    const float s = 1.0f / (1.0f + __expf(-g));
    if (act == 1) {
        slope = s * (1.0f - s);
        return s;
    }
    slope = s * (1.0f + g * (1.0f - s));
    return g * s;
}

template <typename T, int TPR, int V>
__global__ void __launch_bounds__(TPR < 0 ? 1024 : kGroup) k_gated_norm_fwd(GatedNorm p) {
    __shared__ float shared[TPR <= 0 ? 32 : 1];
    const int lanes = TPR <= 0 ? static_cast<int>(blockDim.x) : TPR, groups = static_cast<int>(blockDim.x) / lanes;
    const int lane = threadIdx.x % lanes, group = threadIdx.x / lanes;
    float w[kElems], b[kElems], s[kElems], w2[kElems], b2[kElems];
    load_param<V>(w, p.weight, p.param_type, 1.0f, lane, lanes, p.c);
    load_param<V>(b, p.bias, p.param_type, 0.0f, lane, lanes, p.c);
    load_param<V>(s, p.scale, p.param_type, 1.0f, lane, lanes, p.c);
    load_param<V>(w2, p.next_weight, p.param_type, 1.0f, lane, lanes, p.c);
    load_param<V>(b2, p.next_bias, p.param_type, 0.0f, lane, lanes, p.c);
    // whole blocks stay in the loop: the shuffles name every lane
    for (int64_t row0 = static_cast<int64_t>(blockIdx.x) * groups; row0 < p.rows; row0 += static_cast<int64_t>(gridDim.x) * groups) {
        const int64_t row = row0 + group;
        const bool live = row < p.rows;
        const int c = live ? p.c : 0;
        float x[kElems], h[kElems], g[kElems];
        load_row<T, V>(h, static_cast<const T*>(p.h) + (live ? row * p.h_st : 0), lane, lanes, c);
        load_row<T, V>(x, static_cast<const T*>(p.x) + (live ? row * p.x_st : 0), lane, lanes, c);
        if (p.gate_kind == 2) {
            load_row<T, V>(g, static_cast<const T*>(p.gate) + (live ? row * p.g_st : 0), lane, lanes, c);
        } else {
            const float one = p.gate_kind == 1 && live ? up(static_cast<const T*>(p.gate)[row * p.g_st]) : 1.0f;
#pragma unroll
            for (int i = 0; i < kElems; ++i) g[i] = one;
        }
        const float2 st1 = row_stats<TPR, V>(h, p, lane, lanes, shared);
#pragma unroll
        for (int i = 0; i < kElems; ++i) {
            float slope;
            const float a = p.gate_kind == 0 ? 1.0f : gate_value(g[i], p.act, slope);
            x[i] += s[i] * a * ((h[i] - st1.x) * st1.y * w[i] + b[i]);
        }
        store_row<T, V>(static_cast<T*>(p.y) + (live ? row * p.c : 0), x, lane, lanes, c);
        float2 st2 = make_float2(0.0f, 0.0f);
        if (p.z != nullptr) {
            st2 = row_stats<TPR, V>(x, p, lane, lanes, shared);
#pragma unroll
            for (int i = 0; i < kElems; ++i) x[i] = (x[i] - st2.x) * st2.y * w2[i] + b2[i];
            store_row<T, V>(static_cast<T*>(p.z) + (live ? row * p.c : 0), x, lane, lanes, c);
        }
        if (p.stats != nullptr && live && lane == 0) p.stats[row] = make_float4(st1.x, st1.y, st2.x, st2.y);
    }
}

template <typename T, int TPR, int V>
__global__ void __launch_bounds__(TPR < 0 ? 1024 : kGroup) k_gated_norm_bwd(GatedNorm p) {
    __shared__ float shared[TPR <= 0 ? 96 : 1];
    const int lanes = TPR <= 0 ? static_cast<int>(blockDim.x) : TPR, groups = static_cast<int>(blockDim.x) / lanes;
    const int lane = threadIdx.x % lanes, group = threadIdx.x / lanes;
    float w[kElems], b[kElems], s[kElems], w2[kElems];
    load_param<V>(w, p.weight, p.param_type, 1.0f, lane, lanes, p.c);
    load_param<V>(b, p.bias, p.param_type, 0.0f, lane, lanes, p.c);
    load_param<V>(s, p.scale, p.param_type, 1.0f, lane, lanes, p.c);
    load_param<V>(w2, p.next_weight, p.param_type, 1.0f, lane, lanes, p.c);
    float dw[kElems] = {}, db[kElems] = {}, ds[kElems] = {}, dw2[kElems] = {}, db2[kElems] = {};
    for (int64_t row0 = static_cast<int64_t>(blockIdx.x) * groups; row0 < p.rows; row0 += static_cast<int64_t>(gridDim.x) * groups) {
        const int64_t row = row0 + group;
        const bool live = row < p.rows;
        const int c = live ? p.c : 0;
        float n[kElems], y[kElems], g[kElems], d[kElems];
        load_row<T, V>(n, static_cast<const T*>(p.h) + (live ? row * p.h_st : 0), lane, lanes, c);
        load_row<T, V>(y, static_cast<const T*>(p.x) + (live ? row * p.x_st : 0), lane, lanes, c);
        if (p.gate_kind == 2) {
            load_row<T, V>(g, static_cast<const T*>(p.gate) + (live ? row * p.g_st : 0), lane, lanes, c);
        } else {
            const float one = p.gate_kind == 1 && live ? up(static_cast<const T*>(p.gate)[row * p.g_st]) : 1.0f;
#pragma unroll
            for (int i = 0; i < kElems; ++i) g[i] = one;
        }
        const float4 st = live ? p.stats[row] : make_float4(0.f, 0.f, 0.f, 0.f);
        // y again, then its norm, from the forward's statistics
#pragma unroll
        for (int i = 0; i < kElems; ++i) {
            float slope;
            const float a = p.gate_kind == 0 ? 1.0f : gate_value(g[i], p.act, slope);
            n[i] = (n[i] - st.x) * st.y;
            y[i] += s[i] * a * (n[i] * w[i] + b[i]);
        }
        if (p.dz != nullptr) {
            float u[kElems];
            load_row<T, V>(u, static_cast<const T*>(p.dz) + (live ? row * p.dz_st : 0), lane, lanes, c);
            float m[2] = {0.0f, 0.0f};
#pragma unroll
            for (int i = 0; i < kElems; ++i) {
                y[i] = (y[i] - st.z) * st.w;  // absent columns: u is 0
                dw2[i] = fmaf(u[i], y[i], dw2[i]);
                db2[i] += u[i];
                u[i] *= w2[i];
                m[0] = fmaf(u[i], y[i], m[0]);
                m[1] += u[i];
            }
            row_sum<TPR>(m, shared);
            m[0] *= p.inv_c;
            m[1] = p.layer ? m[1] * p.inv_c : 0.0f;
#pragma unroll
            for (int i = 0; i < kElems; ++i) d[i] = (u[i] - y[i] * m[0] - m[1]) * st.w;
        } else {
#pragma unroll
            for (int i = 0; i < kElems; ++i) d[i] = 0.0f;
        }
        if (p.dy != nullptr) {
            float u[kElems];
            load_row<T, V>(u, static_cast<const T*>(p.dy) + (live ? row * p.dy_st : 0), lane, lanes, c);
#pragma unroll
            for (int i = 0; i < kElems; ++i) d[i] += u[i];
        }
        if (p.dx != nullptr) store_row<T, V>(static_cast<T*>(p.dx) + (live ? row * p.c : 0), d, lane, lanes, c);
        float m[3] = {0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int i = 0; i < kElems; ++i) {
            if (col_of<V>(lane, lanes, i) >= c) d[i] = 0.0f;
            float slope = 0.0f;
            const float a = p.gate_kind == 0 ? 1.0f : gate_value(g[i], p.act, slope);
            const float t = n[i] * w[i] + b[i];
            const float da = d[i] * s[i] * t * slope;
            ds[i] = fmaf(d[i] * a, t, ds[i]);
            d[i] *= s[i] * a;  // dn
            dw[i] = fmaf(d[i], n[i], dw[i]);
            db[i] += d[i];
            d[i] *= w[i];
            m[0] = fmaf(d[i], n[i], m[0]);
            m[1] += d[i];
            m[2] += da;
            g[i] = da;
        }
        row_sum<TPR>(m, shared);
        if (p.dgate != nullptr) {
            if (p.gate_kind == 2)
                store_row<T, V>(static_cast<T*>(p.dgate) + (live ? row * p.c : 0), g, lane, lanes, c);
            else if (live && lane == 0)
                down(static_cast<T*>(p.dgate)[row], m[2]);
        }
        if (p.dh != nullptr) {
            m[0] *= p.inv_c;
            m[1] = p.layer ? m[1] * p.inv_c : 0.0f;
#pragma unroll
            for (int i = 0; i < kElems; ++i) d[i] = (d[i] - n[i] * m[0] - m[1]) * st.y;
            store_row<T, V>(static_cast<T*>(p.dh) + (live ? row * p.c : 0), d, lane, lanes, c);
        }
    }
    // a row of partial sums for each group: [5][gridDim.x groups][c]
    const int64_t part = static_cast<int64_t>(blockIdx.x) * groups + group, parts = static_cast<int64_t>(gridDim.x) * groups;
#pragma unroll
    for (int i = 0; i < kElems; ++i) {
        const int col = col_of<V>(lane, lanes, i);
        if (col >= p.c) continue;
        p.partial[(0 * parts + part) * p.c + col] = dw[i];
        p.partial[(1 * parts + part) * p.c + col] = ds[i];
        p.partial[(2 * parts + part) * p.c + col] = dw2[i];
        if (p.layer) {
            p.partial[(3 * parts + part) * p.c + col] = db[i];
            p.partial[(4 * parts + part) * p.c + col] = db2[i];
        }
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
constexpr int kFwdThreads = 1024, kBwdThreads = 768;

template <typename T, int V>
cudaError_t fwd_vec(const GatedNorm& p, cudaStream_t s) {
    const Shape sh = shape_of(p.rows, p.c, kFwdThreads);
    const unsigned g = static_cast<unsigned>(sh.blocks);
    if (sh.tpr == 8)
        k_gated_norm_fwd<T, 8, V><<<g, sh.threads, 0, s>>>(p);
    else if (sh.tpr == 16)
        k_gated_norm_fwd<T, 16, V><<<g, sh.threads, 0, s>>>(p);
    else if (sh.tpr == 32)
        k_gated_norm_fwd<T, 32, V><<<g, sh.threads, 0, s>>>(p);
    else if (sh.tpr == 0)
        k_gated_norm_fwd<T, 0, V><<<g, sh.threads, 0, s>>>(p);
    else
        k_gated_norm_fwd<T, -1, V><<<g, sh.threads, 0, s>>>(p);
    return cudaGetLastError();
}
template <typename T, int V>
cudaError_t bwd_vec(const GatedNorm& p, cudaStream_t s) {
    const Shape sh = shape_of(p.rows, p.c, kBwdThreads);
    const unsigned g = static_cast<unsigned>(sh.blocks);
    if (sh.tpr == 8)
        k_gated_norm_bwd<T, 8, V><<<g, sh.threads, 0, s>>>(p);
    else if (sh.tpr == 16)
        k_gated_norm_bwd<T, 16, V><<<g, sh.threads, 0, s>>>(p);
    else if (sh.tpr == 32)
        k_gated_norm_bwd<T, 32, V><<<g, sh.threads, 0, s>>>(p);
    else if (sh.tpr == 0)
        k_gated_norm_bwd<T, 0, V><<<g, sh.threads, 0, s>>>(p);
    else
        k_gated_norm_bwd<T, -1, V><<<g, sh.threads, 0, s>>>(p);
    cudaError_t err = cudaGetLastError();
    if (err != cudaSuccess) return err;
    k_gated_norm_reduce<<<dim3((p.c + 31) / 32, p.layer ? 5 : 3), 1024, 0, s>>>(p, sh.blocks * sh.groups);
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
    return 5 * s.blocks * s.groups * c;
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
