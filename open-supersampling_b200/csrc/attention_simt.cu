// Window attention on the FP32 pipe: forward, backward and their small helpers.
//
// Tiles of BM queries x 64 keys. 256 threads as 16 x 16: thread (ty, tx) holds rows ty RM + i and
// keys tx + 16 c of a tile of scores, and rows ty RM + i, columns tx CN + c of an output tile.
// Every product runs on the FP32 pipe from shared memory, 16 RM FMAs for RM + 4 16-byte loads, two
// FMAs an instruction. 510 windows of 64 queries under 144 keys, 4 heads of 32, forward and backward: 693 us (785 us
// with one FMA an instruction and whole tiles at the windows' ends), 12.2 TFLOP/s of 14 dim flops a pair and head where
// the pipe has 74: S and dP are found in both backward kernels, and at 24% of an SM's warps (128 registers) latency
// bounds all three, with half of shared memory's pipe, 45% of the issue slots and 19% of the FP32 pipe taken.
#include "attention.cuh"
#include "internal.h"

namespace oss {
namespace {

constexpr int kThreads = 256;
constexpr int kKeys = 64;  // keys of a tile

// ---- shared-memory layout ---------------------------------------------------
struct Smem {
    float* base;
    __device__ float* take(int n) {
        float* p = base;
        base += (n + 3) & ~3;
        return p;
    }
};

// Rows [first, first + valid) of a packed operand, zeros beyond them and beyond dim.
// row r is token r / pack, head head0 + r % pack.
template <typename T, int DP, int ROWS>
__device__ __forceinline__ void load_rows(float* dst, const void* src, int64_t st, int64_t sh, int64_t token0, int head0,
                                          int pack, int first, int valid, int dim) {
    const T* p = static_cast<const T*>(src);
    constexpr int V = 4;
    const bool vec = sizeof(T) == 4 && dim % V == 0 && st % V == 0 && sh % V == 0 && (reinterpret_cast<uintptr_t>(p) & 15) == 0;
    for (int i = threadIdx.x; i < ROWS * (DP / V); i += kThreads) {
        const int r = i / (DP / V), c = (i % (DP / V)) * V;
        float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
        if (r < valid && c < dim) {
            const int64_t row = first + r;
            const T* q = p + (token0 + row / pack) * st + (head0 + static_cast<int>(row % pack)) * sh + c;
            if (vec) {
                x = __ldg(reinterpret_cast<const float4*>(q));
            } else {
                x.x = to_f(q[0]);
                if (c + 1 < dim) x.y = to_f(q[1]);
                if (c + 2 < dim) x.z = to_f(q[2]);
                if (c + 3 < dim) x.w = to_f(q[3]);
            }
        }
        *reinterpret_cast<float4*>(dst + r * (DP + 4) + c) = x;
    }
}

// acc[i][c] = A[ty RM + i] . B[tx + 16 c] over DP for c < NC: even and odd columns are two sums, so
// that one instruction does both.
template <int DP, int RM, int NC>
__device__ __forceinline__ void dot_cols(float (&acc)[RM][4], const float* A, const float* B, int ty, int tx) {
    constexpr int LD = DP + 4;
    float2 t[RM][NC] = {};
#pragma unroll 4
    for (int d = 0; d < DP; d += 4) {
        float4 a[RM], b[NC];
#pragma unroll
        for (int i = 0; i < RM; ++i) a[i] = *reinterpret_cast<const float4*>(A + (ty * RM + i) * LD + d);
#pragma unroll
        for (int c = 0; c < NC; ++c) b[c] = *reinterpret_cast<const float4*>(B + (tx + 16 * c) * LD + d);
#pragma unroll
        for (int i = 0; i < RM; ++i)
#pragma unroll
            for (int c = 0; c < NC; ++c) {
                t[i][c] = __ffma2_rn(make_float2(a[i].x, a[i].y), make_float2(b[c].x, b[c].y), t[i][c]);
                t[i][c] = __ffma2_rn(make_float2(a[i].z, a[i].w), make_float2(b[c].z, b[c].w), t[i][c]);
            }
    }
#pragma unroll
    for (int i = 0; i < RM; ++i)
#pragma unroll
        for (int c = 0; c < 4; ++c) acc[i][c] = c < NC ? t[i][c < NC ? c : 0].x + t[i][c < NC ? c : 0].y : 0.0f;
}
// The same for the first n rows of B (the others' products are 0): 16 of them at a time.
template <int DP, int RM>
__device__ __forceinline__ void dot_rows(float (&acc)[RM][4], const float* A, const float* B, int n, int ty, int tx) {
    if (n > 48)
        dot_cols<DP, RM, 4>(acc, A, B, ty, tx);
    else if (n > 32)
        dot_cols<DP, RM, 3>(acc, A, B, ty, tx);
    else if (n > 16)
        dot_cols<DP, RM, 2>(acc, A, B, ty, tx);
    else
        dot_cols<DP, RM, 1>(acc, A, B, ty, tx);
}

// acc[i][c] += sum_j P[ty RM + i][j] V[j][tx CN + c], j < n. MASKED: a zero weight takes
// nothing from its row, whatever stands there (a NaN behind a mask stays there).
template <int DP, int RM, int CN, bool MASKED>
__device__ __forceinline__ void weigh_rows(float (&acc)[RM][CN], const float* P, int ldp, const float* V, int n, int ty, int tx) {
    constexpr int LD = DP + 4;
#pragma unroll 2
    for (int j = 0; j < n; j += 4) {
        float4 w[RM];
#pragma unroll
        for (int i = 0; i < RM; ++i) w[i] = *reinterpret_cast<const float4*>(P + (ty * RM + i) * ldp + j);
#pragma unroll
        for (int jj = 0; jj < 4; ++jj) {
            float v[CN];
            if constexpr (CN == 2) {
                const float2 t = *reinterpret_cast<const float2*>(V + (j + jj) * LD + tx * 2);
                v[0] = t.x, v[1] = t.y;
            } else {
#pragma unroll
                for (int n4 = 0; n4 < CN / 4; ++n4) {
                    const float4 t = *reinterpret_cast<const float4*>(V + (j + jj) * LD + n4 * 64 + tx * 4);
                    v[4 * n4] = t.x, v[4 * n4 + 1] = t.y, v[4 * n4 + 2] = t.z, v[4 * n4 + 3] = t.w;
                }
            }
#pragma unroll
            for (int i = 0; i < RM; ++i) {
                const float p = jj == 0 ? w[i].x : jj == 1 ? w[i].y : jj == 2 ? w[i].z : w[i].w;
#pragma unroll
                for (int c = 0; c < CN; c += 2) {
                    const float2 x = make_float2(MASKED && p == 0.0f ? 0.0f : v[c], MASKED && p == 0.0f ? 0.0f : v[c + 1]);
                    const float2 y = __ffma2_rn(make_float2(p, p), x, make_float2(acc[i][c], acc[i][c + 1]));
                    acc[i][c] = y.x;
                    acc[i][c + 1] = y.y;
                }
            }
        }
    }
}

// Column of an output tile that acc[.][c] holds.
template <int CN>
__device__ __forceinline__ int out_col(int tx, int c) {
    return CN <= 2 ? tx * CN + c : (c / 4) * 64 + tx * 4 + (c & 3);
}

// ---- forward -----------------------------------------------------------------
// One pass over the keys with the running maximum and sum of each row.
template <typename T, int DP, int RM>
__global__ void __launch_bounds__(kThreads) k_attn_fwd(AttnParams p) {
    constexpr int BM = 16 * RM, LD = DP + 4, CN = DP / 16, LDP = kKeys + 4;
    extern __shared__ __align__(16) float smem_f[];
    Smem sm{smem_f};
    float* Qs = sm.take(BM * LD);
    float* Ks = sm.take(kKeys * LD);
    float* Vs = sm.take(kKeys * LD);
    float* Ps = sm.take(BM * LDP);
    int2* qpos = reinterpret_cast<int2*>(sm.take(BM * 2));
    int2* kpos = reinterpret_cast<int2*>(sm.take(kKeys * 2));
    const int entries = bias_entries(p.bias);
    float* Es = sm.take(entries * p.pack);
    const int tid = threadIdx.x, tx = tid & 15, ty = tid >> 4;
    const int head0 = blockIdx.y * p.pack, kvh = head0 / (p.heads / p.kv_heads);

    AttnTile t;
    if (!attn_tile(p.q_off, p.tq, p.k_off, p.tk, p.windows, p.pack, BM, blockIdx.x, t)) return;
    const int rows = min(BM, t.len * p.pack - t.first);

    const float c2 = p.scale * kLog2e;
    for (int e = tid; e < entries * p.pack; e += kThreads) Es[e] = bias_entry(p.bias, p.heads, head0 + e / entries, e % entries);
    if (entries > 0)
        for (int r = tid; r < rows; r += kThreads) qpos[r] = bias_pos(p.bias.q_pos, p.bias.axes, t.begin + (t.first + r) / p.pack);
    load_rows<T, DP, BM>(Qs, p.q, p.q_st, p.q_sh, t.begin, head0, p.pack, t.first, rows, p.dim);

    int see[RM];  // keys that each row sees
    int most = 0;
    for (int i = 0; i < RM; ++i) {
        const int r = ty * RM + i;
        see[i] = r >= rows ? 0 : p.causal ? min(max((t.first + r) / p.pack + t.olen - t.len + 1, 0), t.olen) : t.olen;
    }
    most = p.causal ? min(max((t.first + rows - 1) / p.pack + t.olen - t.len + 1, 0), t.olen) : t.olen;
    const int tiles = (most + kKeys - 1) / kKeys;
    const int per = (tiles + p.splits - 1) / p.splits;
    const int tile0 = min(static_cast<int>(blockIdx.z) * per, tiles), tile1 = min(tile0 + per, tiles);

    float o[RM][CN] = {}, m[RM], l[RM];
    for (int i = 0; i < RM; ++i) m[i] = -INFINITY, l[i] = 0.0f;
    for (int kt = tile0; kt < tile1; ++kt) {
        const int k0 = kt * kKeys, n = min(kKeys, t.olen - k0);
        __syncthreads();
        load_rows<T, DP, kKeys>(Ks, p.k, p.k_st, p.k_sh, t.obegin, kvh, 1, k0, n, p.dim);
        load_rows<T, DP, kKeys>(Vs, p.v, p.v_st, p.v_sh, t.obegin, kvh, 1, k0, n, p.dim);
        if (entries > 0 && tid < n) kpos[tid] = bias_pos(p.bias.k_pos, p.bias.axes, t.obegin + k0 + tid);
        __syncthreads();
        float s[RM][4];
        dot_rows<DP, RM>(s, Qs, Ks, n, ty, tx);
        bool cut = false;
#pragma unroll
        for (int i = 0; i < RM; ++i) {
            const int r = ty * RM + i;
            float top = m[i];
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                const int j = tx + 16 * c;
                s[i][c] *= c2;
                if (k0 + j < see[i]) {
                    if (entries > 0) s[i][c] += Es[((t.first + r) % p.pack) * entries + bias_index(p.bias, qpos[r], kpos[j])];
                } else {
                    s[i][c] = -INFINITY;
                    cut = true;
                }
                // a NaN score makes its row NaN, as the formula does: it must not be dropped by the maximum
                top = s[i][c] > top || s[i][c] != s[i][c] ? s[i][c] : top;
            }
#pragma unroll
            for (int x = 1; x < 16; x <<= 1) {
                const float u = __shfl_xor_sync(0xffffffffu, top, x);
                top = u > top || u != u ? u : top;
            }
            const float base = top == -INFINITY ? 0.0f : top;
            const float keep = ex2(m[i] - base);  // 0 before the first visible key
            m[i] = top;
            float sum = 0.0f;
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                s[i][c] = ex2(s[i][c] - base);
                sum += s[i][c];
                Ps[r * LDP + tx + 16 * c] = s[i][c];
            }
#pragma unroll
            for (int x = 1; x < 16; x <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, x);
            l[i] = l[i] * keep + sum;
#pragma unroll
            for (int c = 0; c < CN; ++c) o[i][c] *= keep;
        }
        // every thread takes the same branch
        if (__syncthreads_or(cut))
            weigh_rows<DP, RM, CN, true>(o, Ps, LDP, Vs, n, ty, tx);
        else
            weigh_rows<DP, RM, CN, false>(o, Ps, LDP, Vs, n, ty, tx);
    }
#pragma unroll
    for (int i = 0; i < RM; ++i) {
        const int r = ty * RM + i;
        if (r >= rows) continue;
        const int64_t token = t.begin + (t.first + r) / p.pack;
        const int head = head0 + (t.first + r) % p.pack;
        if (p.splits > 1) {
            const int64_t at = (static_cast<int64_t>(blockIdx.z) * p.tq + token) * p.heads + head;
            if (tx == 0) p.part_ml[2 * at] = m[i], p.part_ml[2 * at + 1] = l[i];
#pragma unroll
            for (int c = 0; c < CN; ++c)
                if (out_col<CN>(tx, c) < p.dim) p.part_o[at * p.dim + out_col<CN>(tx, c)] = o[i][c];
            continue;
        }
        const float inv = l[i] == 0.0f ? 0.0f : 1.0f / l[i];
        T* out = static_cast<T*>(p.out) + (token * p.heads + head) * p.dim;
#pragma unroll
        for (int c = 0; c < CN; ++c)
            if (out_col<CN>(tx, c) < p.dim) out[out_col<CN>(tx, c)] = from_f<T>(o[i][c] * inv);
        if (p.lse != nullptr && tx == 0) store_lse(p, static_cast<int64_t>(head) * p.tq + token, m[i], l[i]);
    }
}

// Joins the parts of a row: o = sum_s o_s 2^(m_s - m) / sum_s l_s 2^(m_s - m). A warp a row.
template <typename T>
__global__ void __launch_bounds__(kThreads) k_attn_join(AttnParams p) {
    const int64_t row = static_cast<int64_t>(blockIdx.x) * (kThreads / 32) + (threadIdx.x >> 5);
    const int lane = threadIdx.x & 31;
    const int64_t rows = static_cast<int64_t>(p.tq) * p.heads;
    if (row >= rows) return;
    float top = -INFINITY;
    for (int s = lane; s < p.splits; s += 32) {
        const float u = p.part_ml[2 * (s * rows + row)];
        top = u > top || u != u ? u : top;
    }
    for (int x = 16; x > 0; x >>= 1) {
        const float u = __shfl_xor_sync(0xffffffffu, top, x);
        top = u > top || u != u ? u : top;
    }
    const float base = top == -INFINITY ? 0.0f : top;
    float l = 0.0f, o[kMaxHeadDim / 32] = {};
    for (int s = 0; s < p.splits; ++s) {
        const int64_t at = s * rows + row;
        const float ls = p.part_ml[2 * at + 1];
        if (ls == 0.0f) continue;  // a part without a visible key
        const float w = ex2(p.part_ml[2 * at] - base);
        l += w * ls;
#pragma unroll
        for (int c = 0; c < kMaxHeadDim / 32; ++c)
            if (lane + 32 * c < p.dim) o[c] = fmaf(w, p.part_o[at * p.dim + lane + 32 * c], o[c]);
    }
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    T* out = static_cast<T*>(p.out) + row * p.dim;
#pragma unroll
    for (int c = 0; c < kMaxHeadDim / 32; ++c)
        if (lane + 32 * c < p.dim) out[lane + 32 * c] = from_f<T>(o[c] * inv);
    if (p.out_lo != nullptr) {
        T* lo = static_cast<T*>(p.out_lo) + row * p.dim;
#pragma unroll
        for (int c = 0; c < kMaxHeadDim / 32; ++c)
            if (lane + 32 * c < p.dim) lo[lane + 32 * c] = from_f<T>(lost_by<T>(o[c] * inv));
    }
    if (p.lse != nullptr && lane == 0) store_lse(p, (row % p.heads) * p.tq + row / p.heads, top, l);
}

// Of 64 bits where it must be: such a division costs some ninety instructions more.
__device__ __forceinline__ int64_t divide(int64_t x, int by) {
    return x >> 32 == 0 ? static_cast<int64_t>(static_cast<uint32_t>(x) / static_cast<uint32_t>(by)) : x / by;
}


// ---- backward ----------------------------------------------------------------
// delta[h][i] = dout . out of a row. LANES lanes a row, two values at a time where its
// address and strides allow it (PAIRS). Bound by the latency of its loads: 13 us for 34560 rows of
// 6 heads of 30.
template <typename T, int LANES, bool PAIRS>
__global__ void __launch_bounds__(kThreads) k_attn_delta(AttnParams p) {
    if ((*p.flags & kSomeLong) == 0) return;  // short windows find their own
    constexpr int V = PAIRS ? 2 : 1;
    struct alignas(V * sizeof(T)) Pair {
        T v[V];
    };
    const int lane = threadIdx.x % LANES;
    const int64_t rows = static_cast<int64_t>(p.tq) * p.heads;
    const int64_t per = kThreads / LANES, step = static_cast<int64_t>(gridDim.x) * per;
    // whole warps stay in the loop: the shuffles name every lane
    for (int64_t row0 = static_cast<int64_t>(blockIdx.x) * per; row0 < rows; row0 += step) {
        const int64_t row = row0 + threadIdx.x / LANES;
        float sum = 0.0f;
        int64_t token = 0, head = 0;
        if (row < rows) {
            token = divide(row, p.heads), head = row - token * p.heads;
            const T* g = static_cast<const T*>(p.dout) + token * p.do_st + head * p.do_sh;
            const T* o = static_cast<const T*>(p.out) + row * p.dim;
            const T* lo = p.out_lo == nullptr ? nullptr : static_cast<const T*>(p.out_lo) + row * p.dim;
            for (int c = V * lane; c < p.dim; c += V * LANES) {
                const Pair x = *reinterpret_cast<const Pair*>(g + c), y = *reinterpret_cast<const Pair*>(o + c);
                Pair less{};
                if (lo != nullptr) less = *reinterpret_cast<const Pair*>(lo + c);
#pragma unroll
                for (int i = 0; i < V; ++i)
                    sum = fmaf(to_f(x.v[i]), to_f(y.v[i]) + (lo == nullptr ? 0.0f : to_f(less.v[i])), sum);
            }
        }
#pragma unroll
        for (int x = LANES / 2; x > 0; x >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, x);
        if (lane == 0 && row < rows) p.delta[head * p.tq + token] = sum;
    }
}

// The weights and their gradients of one 64 x 64 tile, from its scores and dp.
// s: q.k on entry, p on exit; dp: do.v on entry, ds on exit. Zero where the mask is.
template <int RM>
__device__ __forceinline__ bool score_grads(const AttnParams& p, float (&s)[RM][4], float (&dp)[RM][4], int first, int rows,
                                            const AttnTile& w, bool by_query, int k0, int n, const float* lse,
                                            const float* delta, const float* far, const float* Es, int entries, const int2* qpos,
                                            const int2* kpos, int ty, int tx) {
    const int qlen = by_query ? w.len : w.olen, klen = by_query ? w.olen : w.len;
    const float c2 = p.scale * kLog2e;
    bool cut = false;
#pragma unroll
    for (int i = 0; i < RM; ++i) {
        const int r = ty * RM + i;
        const int see = r >= rows ? 0 : p.causal ? min(max(first + r + klen - qlen + 1, 0), klen) : klen;
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            const int j = tx + 16 * c;
            if (j < n && k0 + j < see) {
                float x = s[i][c] * c2;
                if (entries > 0) x += Es[bias_index(p.bias, qpos[r], kpos[j])];
                const float w2 = ex2(x - lse[r]) * far[r];
                s[i][c] = w2;
                dp[i][c] = w2 * (dp[i][c] - delta[r]);
            } else {
                s[i][c] = dp[i][c] = 0.0f;
                cut = true;
            }
        }
    }
    return cut;
}

// dq: a tile of queries walks its window's keys; the bias gradient is summed here too.
// GRAD_BIAS: a block keeps its head and walks slots blockIdx.x, + gridDim.x, .... A tile's terms are
// summed in 64-bit integers at 2^-60 of their sum of magnitudes, then join the block's fp64 sums,
// each by its entry's own thread; those stay in shared memory (`own_acc`), or where a large map leaves no
// room for them in the block's part of p.bias_part.
template <typename T, int DP, bool GRAD_BIAS>
__global__ void __launch_bounds__(kThreads) k_attn_dq(AttnParams p, int own_acc) {
    constexpr int RM = 4, BM = 64, LD = DP + 4, CN = DP / 16, LDP = kKeys + 4;
    extern __shared__ __align__(16) float smem_f[];
    Smem sm{smem_f};
    float* Qs = sm.take(BM * LD);
    float* Gs = sm.take(BM * LD);
    float* Ks = sm.take(kKeys * LD);
    float* Vs = sm.take(kKeys * LD);
    float* Ds = sm.take(BM * LDP);
    float* lse = sm.take(BM);
    float* delta = sm.take(BM);
    float* far = sm.take(BM);
    int2* qpos = reinterpret_cast<int2*>(sm.take(BM * 2));
    int2* kpos = reinterpret_cast<int2*>(sm.take(kKeys * 2));
    const int entries = bias_entries(p.bias);
    float* Es = sm.take(entries);
    uint32_t* lo = reinterpret_cast<uint32_t*>(sm.take(GRAD_BIAS ? entries : 0));
    uint32_t* hi = reinterpret_cast<uint32_t*>(sm.take(GRAD_BIAS ? entries : 0));
    float* wsize = sm.take(GRAD_BIAS ? 8 : 0);
    const int tid = threadIdx.x, tx = tid & 15, ty = tid >> 4;
    const int head = blockIdx.y, kvh = head / (p.heads / p.kv_heads);
    const int slots = attn_slots(p.tq, p.windows, BM);
    double* part = GRAD_BIAS ? p.bias_part + (static_cast<int64_t>(head) * p.bias_parts + blockIdx.x) * entries : nullptr;
    double* acc = GRAD_BIAS && own_acc ? reinterpret_cast<double*>(sm.take(2 * entries)) : part;
    float fixed = 0.0f;  // of the sums that have not joined yet
    if (GRAD_BIAS)
        for (int e = tid; e < entries; e += kThreads) lo[e] = hi[e] = 0u, acc[e] = 0.0;
    auto join = [&] {  // after a barrier
        if (fixed == 0.0f) return;
        const double unit = 1.0 / static_cast<double>(fixed);
        for (int e = tid; e < entries; e += kThreads) {
            const long long sum = static_cast<long long>((static_cast<unsigned long long>(hi[e]) << 32) | lo[e]);
            if (sum != 0) acc[e] += static_cast<double>(sum) * unit, lo[e] = hi[e] = 0u;
        }
        fixed = 0.0f;
    };
    for (int e = tid; e < entries; e += kThreads) Es[e] = bias_entry(p.bias, p.heads, head, e);

    for (int slot = blockIdx.x; slot < slots; slot += gridDim.x) {
        AttnTile t;
        if (!attn_tile(p.q_off, p.tq, p.k_off, p.tk, p.windows, 1, BM, slot, t)) continue;
        const int rows = min(BM, t.len - t.first);
        __syncthreads();
        load_rows<T, DP, BM>(Qs, p.q, p.q_st, p.q_sh, t.begin, head, 1, t.first, rows, p.dim);
        load_rows<T, DP, BM>(Gs, p.dout, p.do_st, p.do_sh, t.begin, head, 1, t.first, rows, p.dim);
        for (int r = tid; r < rows; r += kThreads) {
            const int64_t at = static_cast<int64_t>(head) * p.tq + t.begin + t.first + r;
            lse[r] = p.lse[at], far[r] = far_factor(p, at, lse[r]);
            if (entries > 0) qpos[r] = bias_pos(p.bias.q_pos, p.bias.axes, t.begin + t.first + r);
        }
        __syncthreads();
        // delta = dout . out of the rows, for the kernel of dk and dv as well
#pragma unroll
        for (int i = 0; i < RM; ++i) {
            const int r = ty * RM + i;
            float sum = 0.0f;
            if (r < rows) {
                const T* out = static_cast<const T*>(p.out) + (static_cast<int64_t>(t.begin + t.first + r) * p.heads + head) * p.dim;
#pragma unroll
                for (int c = 0; c < CN; ++c) {
                    const int col = out_col<CN>(tx, c);
                    if (col < p.dim) sum = fmaf(Gs[r * LD + col], to_f(out[col]), sum);
                }
            }
#pragma unroll
            for (int x = 1; x < 16; x <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, x);
            if (tx == 0 && r < rows) {
                delta[r] = sum;
                p.delta[static_cast<int64_t>(head) * p.tq + t.begin + t.first + r] = sum;
            }
        }
        const int most = p.causal ? min(max(t.first + rows + t.olen - t.len, 0), t.olen) : t.olen;
        float dq[RM][CN] = {};
        for (int k0 = 0; k0 < most; k0 += kKeys) {
            const int n = min(kKeys, t.olen - k0);
            __syncthreads();
            if (GRAD_BIAS) join();
            load_rows<T, DP, kKeys>(Ks, p.k, p.k_st, p.k_sh, t.obegin, kvh, 1, k0, n, p.dim);
            load_rows<T, DP, kKeys>(Vs, p.v, p.v_st, p.v_sh, t.obegin, kvh, 1, k0, n, p.dim);
            if (entries > 0 && tid < n) kpos[tid] = bias_pos(p.bias.k_pos, p.bias.axes, t.obegin + k0 + tid);
            __syncthreads();
            float s[RM][4], dp[RM][4];
            dot_rows<DP, RM>(s, Qs, Ks, n, ty, tx);
            dot_rows<DP, RM>(dp, Gs, Vs, n, ty, tx);
            const bool cut = score_grads<RM>(p, s, dp, t.first, rows, t, true, k0, n, lse, delta, far, Es, entries, qpos, kpos, ty, tx);
#pragma unroll
            for (int i = 0; i < RM; ++i)
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    const int r = ty * RM + i, j = tx + 16 * c;
                    Ds[r * LDP + j] = dp[i][c];
                }
            if (GRAD_BIAS) {
                float flat[4 * RM];
#pragma unroll
                for (int i = 0; i < 4 * RM; ++i) flat[i] = dp[i / 4][i % 4];
                const float m = fabsf(warp_size(flat));
                if ((tid & 31) == 0) wsize[tid >> 5] = m;
            }
            const bool masked = __syncthreads_or(cut);
            if (GRAD_BIAS) {
                float m = 0.0f;
                for (int w = 0; w < kThreads / 32; ++w) m += wsize[w];
                fixed = bias_scale(m, 60);
#pragma unroll
                for (int i = 0; i < RM; ++i)
#pragma unroll
                    for (int c = 0; c < 4; ++c) {
                        if (dp[i][c] == 0.0f) continue;
                        const int e = bias_index(p.bias, qpos[ty * RM + i], kpos[tx + 16 * c]);
                        if (is_finite(dp[i][c]))
                            bias_add_shared(lo, hi, e, __float2ll_rn(dp[i][c] * fixed));
                        else
                            bias_mark_bad(p, head, e);
                    }
            }
            if (masked)
                weigh_rows<DP, RM, CN, true>(dq, Ds, LDP, Ks, n, ty, tx);
            else
                weigh_rows<DP, RM, CN, false>(dq, Ds, LDP, Ks, n, ty, tx);
        }
#pragma unroll
        for (int i = 0; i < RM; ++i) {
            const int r = ty * RM + i;
            if (r >= rows) continue;
            T* out = static_cast<T*>(p.dq) + (static_cast<int64_t>(t.begin + t.first + r) * p.heads + head) * p.dim;
#pragma unroll
            for (int c = 0; c < CN; ++c)
                if (out_col<CN>(tx, c) < p.dim) out[out_col<CN>(tx, c)] = from_f<T>(dq[i][c] * p.scale);
        }
    }
    if (GRAD_BIAS) {
        __syncthreads();
        join();
        if (own_acc)
            for (int e = tid; e < entries; e += kThreads) part[e] = acc[e];
    }
}

// dk, dv: a tile of keys walks the queries of every head that shares it.
template <typename T, int DP>
__global__ void __launch_bounds__(kThreads) k_attn_dkv(AttnParams p) {
    constexpr int RM = 4, BM = 64, LD = DP + 4, CN = DP / 16, LDP = BM + 4;
    extern __shared__ __align__(16) float smem_f[];
    Smem sm{smem_f};
    float* Ks = sm.take(kKeys * LD);
    float* Vs = sm.take(kKeys * LD);
    float* Qs = sm.take(BM * LD);
    float* Gs = sm.take(BM * LD);
    float* Pt = sm.take(kKeys * LDP);  // p, then ds, transposed
    float* Dt = sm.take(kKeys * LDP);
    float* lse = sm.take(BM);
    float* delta = sm.take(BM);
    float* far = sm.take(BM);
    int2* qpos = reinterpret_cast<int2*>(sm.take(BM * 2));
    int2* kpos = reinterpret_cast<int2*>(sm.take(kKeys * 2));
    const int entries = bias_entries(p.bias);
    float* Es = sm.take(entries);
    const int tid = threadIdx.x, tx = tid & 15, ty = tid >> 4;
    const int kvh = blockIdx.y, group = p.heads / p.kv_heads;

    AttnTile t;
    if (!attn_tile(p.k_off, p.tk, p.q_off, p.tq, p.windows, 1, kKeys, blockIdx.x, t)) return;
    const int n = min(kKeys, t.len - t.first);
    load_rows<T, DP, kKeys>(Ks, p.k, p.k_st, p.k_sh, t.begin, kvh, 1, t.first, n, p.dim);
    load_rows<T, DP, kKeys>(Vs, p.v, p.v_st, p.v_sh, t.begin, kvh, 1, t.first, n, p.dim);
    if (entries > 0 && tid < n) kpos[tid] = bias_pos(p.bias.k_pos, p.bias.axes, t.begin + t.first + tid);
    // the first query that sees this tile's first key
    const int from = p.causal ? max(t.first - (t.len - t.olen), 0) : 0;
    float dk[RM][CN] = {}, dv[RM][CN] = {};
    for (int g = 0; g < group; ++g) {
        const int head = kvh * group + g;
        if (entries > 0) {
            __syncthreads();
            for (int e = tid; e < entries; e += kThreads) Es[e] = bias_entry(p.bias, p.heads, head, e);
        }
        for (int q0 = from / BM * BM; q0 < t.olen; q0 += BM) {
            const int rows = min(BM, t.olen - q0);
            __syncthreads();
            load_rows<T, DP, BM>(Qs, p.q, p.q_st, p.q_sh, t.obegin, head, 1, q0, rows, p.dim);
            load_rows<T, DP, BM>(Gs, p.dout, p.do_st, p.do_sh, t.obegin, head, 1, q0, rows, p.dim);
            for (int r = tid; r < rows; r += kThreads) {
                const int64_t at = static_cast<int64_t>(head) * p.tq + t.obegin + q0 + r;
                lse[r] = p.lse[at], delta[r] = p.delta[at], far[r] = far_factor(p, at, lse[r]);
                if (entries > 0) qpos[r] = bias_pos(p.bias.q_pos, p.bias.axes, t.obegin + q0 + r);
            }
            __syncthreads();
            float s[RM][4], dp[RM][4];
            dot_rows<DP, RM>(s, Qs, Ks, n, ty, tx);
            dot_rows<DP, RM>(dp, Gs, Vs, n, ty, tx);
            const bool cut = score_grads<RM>(p, s, dp, q0, rows, t, false, t.first, n, lse, delta, far, Es, entries, qpos, kpos, ty, tx);
#pragma unroll
            for (int c = 0; c < 4; ++c) {  // RM = 4: a row's four values together
                *reinterpret_cast<float4*>(Pt + (tx + 16 * c) * LDP + ty * RM) = make_float4(s[0][c], s[1][c], s[2][c], s[3][c]);
                *reinterpret_cast<float4*>(Dt + (tx + 16 * c) * LDP + ty * RM) = make_float4(dp[0][c], dp[1][c], dp[2][c], dp[3][c]);
            }
            if (__syncthreads_or(cut)) {
                weigh_rows<DP, RM, CN, true>(dv, Pt, LDP, Gs, rows, ty, tx);
                weigh_rows<DP, RM, CN, true>(dk, Dt, LDP, Qs, rows, ty, tx);
            } else {
                weigh_rows<DP, RM, CN, false>(dv, Pt, LDP, Gs, rows, ty, tx);
                weigh_rows<DP, RM, CN, false>(dk, Dt, LDP, Qs, rows, ty, tx);
            }
        }
    }
#pragma unroll
    for (int i = 0; i < RM; ++i) {
        const int r = ty * RM + i;
        if (r >= n) continue;
        const int64_t at = (static_cast<int64_t>(t.begin + t.first + r) * p.kv_heads + kvh) * p.dim;
#pragma unroll
        for (int c = 0; c < CN; ++c) {
            const int col = out_col<CN>(tx, c);
            if (col >= p.dim) continue;
            static_cast<T*>(p.dk)[at + col] = from_f<T>(dk[i][c] * p.scale);
            static_cast<T*>(p.dv)[at + col] = from_f<T>(dv[i][c]);
        }
    }
}

// ---- the bias gradient of all blocks -----------------------------------------------
// The parts of each entry into the first part: thread (part lane, entry) adds every eighth part, the
// eight sums are added in order.
__global__ void __launch_bounds__(256) k_attn_bias_parts(AttnParams p) {
    __shared__ double sums[8][32];
    const int entries = bias_entries(p.bias), lane = threadIdx.x & 31, row = threadIdx.x >> 5, e = blockIdx.x * 32 + lane;
    const int flags = p.flags == nullptr ? kSomeLong : *p.flags, first_long = p.bias_tiny + p.bias_short;
    double* at = p.bias_part + static_cast<int64_t>(blockIdx.y) * p.bias_parts * entries + e;
    double sum = 0.0;
    if (e < entries) {
        for (int s = row; s < p.bias_parts; s += 8) {
            const bool filled = s < p.bias_tiny || (s < first_long ? (flags & kSomeShort) != 0 : (flags & kSomeLong) != 0);
            if (filled) sum += at[static_cast<int64_t>(s) * entries];
        }
    }
    sums[row][lane] = sum;
    __syncthreads();
    if (row != 0 || e >= entries) return;
    for (int r = 1; r < 8; ++r) sum += sums[r][lane];
    at[0] = sum;
}

// Entries to the rows of the table that they map to: in 64-bit fixed point, so that several
// entries of one row add up the same in any order, at a scale of the row's own (with one for all rows
// of a head, a window of large gradients took the bits of the rows that only others reach). A block a head.
__device__ __forceinline__ int table_shift(unsigned long long top) {
    const double most = __longlong_as_double(static_cast<long long>(top));
    return most > 0.0 ? 48 - ilogb(most) : 0;  // 4096 entries of at most 2^49
}
__global__ void __launch_bounds__(1024) k_attn_bias_table(AttnParams p, void* dtable) {
    const int entries = bias_entries(p.bias), head = blockIdx.x, tid = threadIdx.x;
    const double* sum = p.bias_part + static_cast<int64_t>(head) * p.bias_parts * entries;
    for (int e = tid; e < entries; e += 1024) {
        const int bucket = __ldg(p.bias.map + e);
        if (bucket < 0 || bucket >= p.bias.buckets) continue;
        const int64_t i = static_cast<int64_t>(bucket) * p.heads + head;
        if (isfinite(sum[e]))
            atomicMax(p.bias_top + i, static_cast<unsigned long long>(__double_as_longlong(fabs(sum[e]))));
        else
            p.bias_bad[i] = 1u;
    }
    __threadfence();
    __syncthreads();
    for (int e = tid; e < entries; e += 1024) {
        const int bucket = __ldg(p.bias.map + e);
        if (bucket >= 0 && bucket < p.bias.buckets && isfinite(sum[e])) {
            const int64_t i = static_cast<int64_t>(bucket) * p.heads + head;
            atomicAdd(p.bias_acc + i, static_cast<unsigned long long>(__double2ll_rn(ldexp(sum[e], table_shift(__ldcg(p.bias_top + i))))));
        }
    }
    __threadfence();
    __syncthreads();
    for (int b = tid; b < p.bias.buckets; b += 1024) {
        const int64_t i = static_cast<int64_t>(b) * p.heads + head;
        const double x = ldexp(static_cast<double>(static_cast<long long>(__ldcg(p.bias_acc + i))), -table_shift(__ldcg(p.bias_top + i)));
        store_typed(dtable, p.bias.table_type, i, __ldcg(p.bias_bad + i) ? __uint_as_float(0x7fffffffu) : static_cast<float>(x));
    }
}

int64_t floats(int64_t n) { return (n + 3) / 4 * 4; }

template <typename T, int DP, int RM>
cudaError_t fwd_one(const AttnParams& p, cudaStream_t s) {
    constexpr int BM = 16 * RM;
    const int64_t bytes = 4 * (floats(BM * (DP + 4)) + 2 * floats(kKeys * (DP + 4)) + floats(BM * (kKeys + 4)) + BM * 2 +
                               kKeys * 2 + floats(static_cast<int64_t>(bias_entries(p.bias)) * p.pack));
    cudaError_t err = allow_smem(k_attn_fwd<T, DP, RM>);
    if (err != cudaSuccess) return err;
    const dim3 grid(attn_slots(static_cast<int64_t>(p.tq) * p.pack, p.windows, BM), p.heads / p.pack, p.splits);
    k_attn_fwd<T, DP, RM><<<grid, kThreads, bytes, s>>>(p);
    return cudaGetLastError();
}

template <typename T, int DP>
cudaError_t fwd_rows(const AttnParams& p, cudaStream_t s) {
    // Tiles of 16 rows where the average window has no more: a quarter of the work on empty rows.
    return static_cast<int64_t>(p.tq) * p.pack <= 16ll * p.windows ? fwd_one<T, DP, 1>(p, s) : fwd_one<T, DP, 4>(p, s);
}

cudaError_t fwd_f32(const AttnParams& p, cudaStream_t s) {
    return p.dim <= 32 ? fwd_rows<float, 32>(p, s) : p.dim <= 64 ? fwd_rows<float, 64>(p, s) : fwd_rows<float, 128>(p, s);
}

template <typename T>
cudaError_t join_parts(const AttnParams& p, cudaStream_t s) {
    const int64_t rows = static_cast<int64_t>(p.tq) * p.heads;
    k_attn_join<T><<<static_cast<unsigned>((rows + 7) / 8), kThreads, 0, s>>>(p);
    return cudaGetLastError();
}

template <typename T, int DP>
cudaError_t bwd_dim(const AttnParams& p, cudaStream_t s) {
    const int64_t entries = bias_entries(p.bias);
    const bool grad_bias = p.bias_part != nullptr;
    int64_t dq_bytes = 4 * (4 * floats(64 * (DP + 4)) + floats(64 * 68) + 3 * 64 + 4 * 64 + floats(entries) * (grad_bias ? 3 : 1) +
                            (grad_bias ? 8 : 0));
    const int own_acc = grad_bias && dq_bytes + 4 * floats(2 * entries) <= kMaxSmem;
    if (own_acc) dq_bytes += 4 * floats(2 * entries);
    const int slots = attn_slots(p.tq, p.windows, 64);
    cudaError_t err;
    if (grad_bias) {
        if ((err = allow_smem(k_attn_dq<T, DP, true>)) != cudaSuccess) return err;
        k_attn_dq<T, DP, true><<<dim3(p.dq_blocks, p.heads), kThreads, dq_bytes, s>>>(p, own_acc);
    } else {
        if ((err = allow_smem(k_attn_dq<T, DP, false>)) != cudaSuccess) return err;
        k_attn_dq<T, DP, false><<<dim3(slots, p.heads), kThreads, dq_bytes, s>>>(p, 0);
    }
    if ((err = cudaGetLastError()) != cudaSuccess) return err;
    const int64_t kv_bytes = 4 * (4 * floats(64 * (DP + 4)) + 2 * floats(64 * 68) + 3 * 64 + 4 * 64 + floats(entries));
    if ((err = allow_smem(k_attn_dkv<T, DP>)) != cudaSuccess) return err;
    k_attn_dkv<T, DP><<<dim3(attn_slots(p.tk, p.windows, kKeys), p.kv_heads), kThreads, kv_bytes, s>>>(p);
    return cudaGetLastError();
}

template <typename T, int LANES>
cudaError_t delta_lanes(const AttnParams& p, cudaStream_t s, int sms) {
    const int64_t blocks = (static_cast<int64_t>(p.tq) * p.heads * LANES + kThreads - 1) / kThreads;
    if (blocks == 0) return cudaSuccess;
    const unsigned grid = static_cast<unsigned>(blocks < 16 * sms ? blocks : 16 * sms);
    const uintptr_t bytes = reinterpret_cast<uintptr_t>(p.dout) | reinterpret_cast<uintptr_t>(p.out) | reinterpret_cast<uintptr_t>(p.out_lo);
    const bool pairs = bytes % (2 * sizeof(T)) == 0 && ((p.do_st | p.do_sh | p.dim) & 1) == 0;
    if (pairs)
        k_attn_delta<T, LANES, true><<<grid, kThreads, 0, s>>>(p);
    else
        k_attn_delta<T, LANES, false><<<grid, kThreads, 0, s>>>(p);
    return cudaGetLastError();
}
template <typename T>
cudaError_t delta_type(const AttnParams& p, cudaStream_t s, int sms) {
    return p.dim <= 32 ? delta_lanes<T, 8>(p, s, sms) : delta_lanes<T, 16>(p, s, sms);
}

}  // namespace

cudaError_t launch_attn_forward(const AttnParams& p, int type, cudaStream_t s) {
    cudaError_t err = cudaSuccess;
    if (p.tiny_max > 0) err = launch_attn_forward_tiny(p, type, s);
    if (err == cudaSuccess) err = type == kF32 ? fwd_f32(p, s) : launch_attn_forward_mma(p, type, s);
    if (err != cudaSuccess || p.splits == 1) return err;
    return type == kF32 ? join_parts<float>(p, s) : type == kBF16 ? join_parts<__nv_bfloat16>(p, s) : join_parts<__half>(p, s);
}

cudaError_t launch_attn_delta(const AttnParams& p, int type, int sms, cudaStream_t s) {
    return type == kBF16 ? delta_type<__nv_bfloat16>(p, s, sms) : delta_type<__half>(p, s, sms);
}

cudaError_t launch_attn_bias_grad(const AttnParams& p, void* dtable, cudaStream_t s) {
    k_attn_bias_parts<<<dim3((bias_entries(p.bias) + 31) / 32, p.heads), 256, 0, s>>>(p);
    const cudaError_t err = cudaGetLastError();
    if (err != cudaSuccess) return err;
    k_attn_bias_table<<<p.heads, 1024, 0, s>>>(p, dtable);
    return cudaGetLastError();
}

cudaError_t launch_attn_backward(const AttnParams& p, int type, void* dtable, int sms, cudaStream_t s) {
    if (type != kF32) return launch_attn_backward_mma(p, type, dtable, sms, s);
    const cudaError_t err = p.dim <= 32 ? bwd_dim<float, 32>(p, s) : p.dim <= 64 ? bwd_dim<float, 64>(p, s) : bwd_dim<float, 128>(p, s);
    return err != cudaSuccess || dtable == nullptr ? err : launch_attn_bias_grad(p, dtable, s);
}

}  // namespace oss
