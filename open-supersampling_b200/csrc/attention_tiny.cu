// Window attention of 16-bit types over few keys: the Gaussians of a tile under all its pixels.
//
// Such windows are bound by reading q (and dout) and writing out (and dq); the products are small
// and a round trip through tensor memory and block barriers costs more than they do. So each
// warp works alone: it holds its window's keys and values in registers as operands of warp-level products
// (m16n8k16) and walks the queries 16 rows at a time, straight from and to global memory.
//
// One register image serves every product. Lane (g, t) = (lane / 4, lane % 4) loads 16 bytes of row
// g: columns 8 t .. 8 t + 7, as registers j = 0 .. 3 of two values.
//   - as operands of q k^T the registers are the k-slots: the same order of columns on both
//     sides, and a sum does not mind which order that is
//   - register j of all lanes is an 8 x 8 block whose column 2 t + i is column 8 t + 2 j + i of the
//     row; transposed in registers it is the right operand of P V, dS K, P^T dO, dS^T Q, and the
//     result's fragment of block j is again columns 8 t + 2 j + i, so that a lane's results of
//     j = 0 .. 3 are 16 consecutive bytes of a row
// P and dS go from accumulators to operands without leaving the lane, transposed in registers
// for P^T and dS^T.
//
// 8160 windows of 256 under 24 keys on average, 4 heads over 2 of 32: 424 us (1217 us by the tcgen05 kernel), of
// which 218 us for up to 32 keys, 102 us for 33 to 64, 67 us for 65 to 128. Latency bounds it: their registers leave
// 11 to 25% of an SM's warps, which wait for loads and for one instruction after the other; half of the issue
// slots (a quarter with 65 keys and more) and 43% of DRAM at most are taken. The backward, 2040 windows under 8 keys
// with a bias gradient: 278 us for up to 16 keys, 78 us for 17 to 32, at 12% of the warps and 28% of the issue slots.
#include "attention_mma.cuh"
#include "internal.h"

namespace oss {
namespace {

constexpr int kWarps = 4;

template <typename T>
__device__ __forceinline__ void mma16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    if constexpr (std::is_same<T, __nv_bfloat16>::value)
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                     : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
    else
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                     : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose8(uint32_t a) {
    uint32_t d;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
    return d;
}

// 8 columns of rows of one operand, DB blocks of 32 columns.
template <typename T, int DB>
struct Rows {
    const T* p;  // the head's columns 8 t ..
    int64_t st;
    int left;    // columns from there to dim
    bool vec, pairs;  // every row starts on 16 bytes and ends on them; on 4
    __device__ __forceinline__ Rows(const void* q, int64_t st_, int64_t sh, int dim, int head) : st(st_) {
        const int t = threadIdx.x & 3;
        p = static_cast<const T*>(q) + head * sh + 8 * t;
        left = dim - 8 * t;
        vec = ((reinterpret_cast<uintptr_t>(q) & 15) | ((st_ | sh | dim) & 7)) == 0;
        pairs = ((reinterpret_cast<uintptr_t>(q) & 3) | ((st_ | sh | dim) & 1)) == 0;
    }
    __device__ __forceinline__ void load(uint32_t (&r)[DB][4], int64_t row, bool live) const { load_at(r, p + row * st, live); }
    // at: column 8 t of the row
    __device__ __forceinline__ void load_at(uint32_t (&r)[DB][4], const T* at, bool live) const {
#pragma unroll
        for (int b = 0; b < DB; ++b) {
#pragma unroll
            for (int j = 0; j < 4; ++j) r[b][j] = 0u;
            const int n = left - 32 * b;
            if (!live || n <= 0) continue;
            const T* from = at + 32 * b;
            if (vec) {
                const uint4 x = __ldg(reinterpret_cast<const uint4*>(from));
                r[b][0] = x.x, r[b][1] = x.y, r[b][2] = x.z, r[b][3] = x.w;
            } else if (pairs) {
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    if (2 * j < n) r[b][j] = __ldg(reinterpret_cast<const uint32_t*>(from) + j);
            } else {
                const unsigned short* s = reinterpret_cast<const unsigned short*>(from);
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    if (e < n) r[b][e >> 1] |= static_cast<uint32_t>(__ldg(s + e)) << (16 * (e & 1));
            }
        }
    }
};

// The accumulators of 8 columns a row, back to a row; h: 0 for row g, 1 for row g + 8.
template <typename T, int DB>
__device__ __forceinline__ void store_row16(T* row, int dim, const float (&o)[DB][4][4], int h, float by) {
    const int t = threadIdx.x & 3;
    const bool vec = dim % 8 == 0 && (reinterpret_cast<uintptr_t>(row) & 15) == 0;
#pragma unroll
    for (int b = 0; b < DB; ++b) {
        const int col = 32 * b + 8 * t;
        if (col >= dim) continue;
        uint32_t w[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) w[j] = pack2(o[b][j][2 * h] * by, o[b][j][2 * h + 1] * by, T{});
        if (vec) {
            *reinterpret_cast<uint4*>(row + col) = make_uint4(w[0], w[1], w[2], w[3]);
        } else if (dim % 2 == 0 && (reinterpret_cast<uintptr_t>(row) & 3) == 0) {
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (col + 2 * j < dim) reinterpret_cast<uint32_t*>(row + col)[j] = w[j];
        } else {
            unsigned short* to = reinterpret_cast<unsigned short*>(row + col);
#pragma unroll
            for (int e = 0; e < 8; ++e)
                if (col + e < dim) to[e] = static_cast<unsigned short>(w[e >> 1] >> (16 * (e & 1)));
        }
    }
}

__device__ __forceinline__ float quad_sum(float x) {
    x += __shfl_xor_sync(0xffffffffu, x, 1);
    return x + __shfl_xor_sync(0xffffffffu, x, 2);
}
__device__ __forceinline__ float quad_max(float x) {
    x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 1));
    return fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 2));
}
__device__ __forceinline__ float warp_sum(float x) {
#pragma unroll
    for (int s = 16; s > 0; s >>= 1) x += __shfl_xor_sync(0xffffffffu, x, s);
    return x;
}

// A warp's window: keys in smem (positions) and where its rows are.
template <int NB>
struct TinyPos {
    int y[8 * NB], x[8 * NB], code[8 * NB];
};

template <int NB>
__device__ __forceinline__ Range tiny_key_pos(TinyPos<NB>* s, const AttnBias& b, int64_t token, int n) {
    const int lane = threadIdx.x & 31;
    Range range{0, 0, 0, 0};
    __syncwarp();
#pragma unroll
    for (int base = 0; base < 8 * NB; base += 32) {  // whole warps: the ranges name every lane
        const int j = base + lane, y0 = bias_pos(b.k_pos, b.axes, token).x;
        const int2 p = bias_pos(b.k_pos, b.axes, token + min(j, n - 1));
        if (j < 8 * NB) {
            s->y[j] = p.x;
            s->x[j] = p.y;
            s->code[j] = linear_code(b, p.x - y0, p.y);
        }
        const Range r = warp_range(p);
        range = base == 0 ? r : join(range, r);
    }
    __syncwarp();
    return range;
}

// Entries of the bias for rows g and g + 8 and keys 8 kb + 2 t + i.
template <int NB>
struct TinyBias {
    const AttnBias& b;
    const TinyPos<NB>* k;
    int2 q[2];
    int off[2];
    bool linear;
    __device__ __forceinline__ TinyBias(const AttnBias& b_, const TinyPos<NB>* k_, const Range& kr, int64_t token, int last, int r0, bool on)
        : b(b_), k(k_), linear(false) {
        if (!on) return;
        const int g = (threadIdx.x & 31) >> 2, y0 = k->y[0];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            q[h] = bias_pos(b.q_pos, b.axes, token + min(r0 + g + 8 * h, last));
            off[h] = linear_code(b, b.ry + y0 - q[h].x, b.rx - q[h].y);
        }
        const Range qr = join(warp_range(q[0]), warp_range(q[1]));
        linear = bias_mode(b, qr, kr) == kLinear;
    }
    __device__ __forceinline__ int entry_linear(int h, int kb, int i) const {
        return off[h] + k->code[8 * kb + 2 * (threadIdx.x & 3) + i];
    }
    __device__ __forceinline__ int entry(int h, int kb, int i) const {
        const int j = 8 * kb + 2 * (threadIdx.x & 3) + i;
        return linear ? off[h] + k->code[j] : bias_index(b, q[h], make_int2(k->y[j], k->x[j]));
    }
};

// Which windows and heads a warp walks: `side` key heads of a block's warps side by side.
struct Share {
    int kvh, first, step;  // key head (may lie past the last one); first window, and the step to the next
};
__device__ __forceinline__ Share share_of(int kv_heads) {
    const int side = kv_heads >= 4 ? 4 : kv_heads >= 2 ? 2 : 1, warp = threadIdx.x >> 5;
    return {static_cast<int>(blockIdx.y) * side + warp % side, static_cast<int>(blockIdx.x) * (kWarps / side) + warp / side,
            static_cast<int>(gridDim.x) * (kWarps / side)};
}

constexpr int tiny_fwd_blocks(int db, int nb) { return nb == 16 ? 2 : db == 1 && nb == 4 ? 4 : 3; }
constexpr int tiny_bwd_blocks(int nb) { return nb == 2 ? 3 : 2; }

// ---- forward --------------------------------------------------------------------------------
// One window and key head, rows [r_begin, r_end), with NK blocks of 8 keys (the lower half of them full).
// The values of 16 blocks do not fit the registers beside their keys: they are loaded again each step.
template <typename T, int DB, int NK, bool BIAS>
__device__ __forceinline__ void tiny_forward(const AttnParams& p, int kvh, int group, int q0, int lq, int k0, int n, int r_begin,
                                             int r_end, TinyPos<NK>* kp, const float* E, int entries) {
    const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const float c2 = p.scale * kLog2e;
    constexpr bool kKeepV = NK <= 8;
    uint32_t kr[NK][DB][4], vt[kKeepV ? NK : 2][DB][4];
    const Rows<T, DB> rv(p.v, p.v_st, p.v_sh, p.dim, kvh);
    {
        const Rows<T, DB> rk(p.k, p.k_st, p.k_sh, p.dim, kvh);
#pragma unroll
        for (int kb = 0; kb < NK; ++kb) {
            rk.load(kr[kb], k0 + 8 * kb + g, 8 * kb + g < n);
            if (kKeepV) rv.load(vt[kKeepV ? kb : 0], k0 + 8 * kb + g, 8 * kb + g < n);
        }
#pragma unroll
        for (int kb = 0; kb < (kKeepV ? NK : 0); ++kb)
#pragma unroll
            for (int b = 0; b < DB; ++b)
#pragma unroll
                for (int j = 0; j < 4; ++j) vt[kb][b][j] = transpose8(vt[kb][b][j]);
    }
    Range krange{0, 0, 0, 0};
    if (BIAS) krange = tiny_key_pos<NK>(kp, p.bias, k0, n);
    const int left = n - 2 * t;  // key 8 kb + 2 t + i is there where 8 kb + i < left
    // Sixteen rows of one head a step, the heads of the group in turn (their rows lie side by side), the
    // loads two steps ahead.
    const Rows<T, DB> rq(p.q, p.q_st, p.q_sh, p.dim, kvh * group);
    uint32_t qa[DB][4], qb[DB][4], na[DB][4], nb[DB][4];
    const T* from = rq.p + static_cast<int64_t>(q0 + r_begin + g) * p.q_st;  // of row g: the next rows to load
    int from_row = r_begin + g, from_head = 0;
    auto fetch = [&](uint32_t (&x)[DB][4], uint32_t (&y)[DB][4]) {
        const T* at = from + from_head * p.q_sh;
        rq.load_at(x, at, from_row < r_end);
        rq.load_at(y, at + 8 * p.q_st, from_row + 8 < r_end);
        if (++from_head == group) from_head = 0, from_row += 16, from += 16 * p.q_st;
    };
    fetch(qa, qb);
    fetch(na, nb);
    T* to_row = static_cast<T*>(p.out) + (static_cast<int64_t>(q0 + r_begin + g) * p.heads + kvh * group) * p.dim;
    const int64_t to_step = static_cast<int64_t>(8) * p.heads * p.dim;
    for (int r0 = r_begin; r0 < r_end; r0 += 16, to_row += 2 * to_step) {
        const TinyBias<NK> tb(p.bias, kp, krange, q0, lq - 1, r0, BIAS);
        for (int gh = 0; gh < group; ++gh) {
            const int head = kvh * group + gh;
            const float* Eh = E + gh * entries;
            T* to = to_row + gh * p.dim;
            float s[NK][4];
#pragma unroll
            for (int kb = 0; kb < NK; ++kb) {
#pragma unroll
                for (int i = 0; i < 4; ++i) s[kb][i] = 0.0f;
#pragma unroll
                for (int b = 0; b < DB; ++b)
#pragma unroll
                    for (int h = 0; h < 2; ++h)
                        mma16<T>(s[kb], qa[b][2 * h], qb[b][2 * h], qa[b][2 * h + 1], qb[b][2 * h + 1], kr[kb][b][2 * h],
                                 kr[kb][b][2 * h + 1]);
            }
#pragma unroll
            for (int b = 0; b < DB; ++b)
#pragma unroll
                for (int j = 0; j < 4; ++j) qa[b][j] = na[b][j], qb[b][j] = nb[b][j];
            fetch(na, nb);
            if (BIAS) {
                if (tb.linear) {
#pragma unroll
                    for (int kb = 0; kb < NK; ++kb)
#pragma unroll
                        for (int i = 0; i < 4; ++i) s[kb][i] = fmaf(s[kb][i], c2, Eh[tb.entry_linear(i >> 1, kb, i & 1)]);
                } else {
#pragma unroll
                    for (int kb = 0; kb < NK; ++kb)
#pragma unroll
                        for (int i = 0; i < 4; ++i) s[kb][i] = fmaf(s[kb][i], c2, Eh[tb.entry(i >> 1, kb, i & 1)]);
                }
            }
#pragma unroll
            for (int kb = NK / 2; kb < NK; ++kb)
#pragma unroll
                for (int i = 0; i < 4; ++i) s[kb][i] = 8 * kb + (i & 1) < left ? s[kb][i] : -INFINITY;
            if (NK == 2) {
#pragma unroll
                for (int i = 0; i < 4; ++i) s[0][i] = (i & 1) < left ? s[0][i] : -INFINITY;
            }
            float2 top = make_float2(-INFINITY, -INFINITY), sum = make_float2(0.0f, 0.0f), off;
#pragma unroll
            for (int kb = 0; kb < NK; ++kb) {
                top.x = fmaxf(top.x, fmaxf(s[kb][0], s[kb][1]));
                top.y = fmaxf(top.y, fmaxf(s[kb][2], s[kb][3]));
            }
            top.x = quad_max(top.x) * (BIAS ? 1.0f : c2);
            top.y = quad_max(top.y) * (BIAS ? 1.0f : c2);
            off.x = top.x == -INFINITY ? 0.0f : -top.x;
            off.y = top.y == -INFINITY ? 0.0f : -top.y;
            const float2 by = make_float2(c2, c2), offx = make_float2(off.x, off.x), offy = make_float2(off.y, off.y);
            float2 sx = make_float2(0.0f, 0.0f), sy = sx;
            uint32_t pk[NK][2];
#pragma unroll
            for (int kb = 0; kb < NK; ++kb) {
                float2 a = make_float2(s[kb][0], s[kb][1]), b = make_float2(s[kb][2], s[kb][3]);
                a = BIAS ? __fadd2_rn(a, offx) : __ffma2_rn(a, by, offx);
                b = BIAS ? __fadd2_rn(b, offy) : __ffma2_rn(b, by, offy);
                a.x = ex2(a.x), a.y = ex2(a.y), b.x = ex2(b.x), b.y = ex2(b.y);
                sx = __fadd2_rn(sx, a);
                sy = __fadd2_rn(sy, b);
                pk[kb][0] = pack2(a.x, a.y, T{});
                pk[kb][1] = pack2(b.x, b.y, T{});
            }
            float o[DB][4][4] = {};
#pragma unroll
            for (int kk = 0; kk < NK / 2; ++kk) {
                const int v0 = kKeepV ? 2 * kk : 0;
                if (!kKeepV) {
                    if (16 * kk >= n) break;
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        rv.load(vt[h], k0 + 16 * kk + 8 * h + g, 16 * kk + 8 * h + g < n);
#pragma unroll
                        for (int b = 0; b < DB; ++b)
#pragma unroll
                            for (int j = 0; j < 4; ++j) vt[h][b][j] = transpose8(vt[h][b][j]);
                    }
                }
#pragma unroll
                for (int b = 0; b < DB; ++b)
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        mma16<T>(o[b][j], pk[2 * kk][0], pk[2 * kk][1], pk[2 * kk + 1][0], pk[2 * kk + 1][1], vt[v0][b][j],
                                 vt[v0 + 1][b][j]);
            }
            sum.x = quad_sum(sx.x + sx.y);
            sum.y = quad_sum(sy.x + sy.y);
            if (r0 + g < r_end) store_row16<T, DB>(to, p.dim, o, 0, sum.x == 0.0f ? 0.0f : __fdividef(1.0f, sum.x));
            if (r0 + g + 8 < r_end) store_row16<T, DB>(to + to_step, p.dim, o, 1, sum.y == 0.0f ? 0.0f : __fdividef(1.0f, sum.y));
            if (NK == 16 && p.out_lo != nullptr) {  // windows of fewer keys find dout . out by themselves
                const float ix = sum.x == 0.0f ? 0.0f : __fdividef(1.0f, sum.x), iy = sum.y == 0.0f ? 0.0f : __fdividef(1.0f, sum.y);
#pragma unroll
                for (int b = 0; b < DB; ++b)
#pragma unroll
                    for (int j = 0; j < 4; ++j)
#pragma unroll
                        for (int i = 0; i < 4; ++i) o[b][j][i] = lost_by<T>(o[b][j][i] * (i < 2 ? ix : iy));
                T* lo = static_cast<T*>(p.out_lo) + (to - static_cast<T*>(p.out));
                if (r0 + g < r_end) store_row16<T, DB>(lo, p.dim, o, 0, 1.0f);
                if (r0 + g + 8 < r_end) store_row16<T, DB>(lo + to_step, p.dim, o, 1, 1.0f);
            }
            if (p.lse != nullptr && t == 0) {
                const int64_t at = static_cast<int64_t>(head) * p.tq + q0 + r0 + g;
                if (r0 + g < r_end) store_lse(p, at, top.x, sum.x);
                if (r0 + g + 8 < r_end) store_lse(p, at + 8, top.y, sum.y);
            }
        }
    }
}

// The walk of the forward kernels: pieces of up to kPiece rows of a window, listed by class (up to 32 keys,
// 33 to 64, 65 to 128) and taken from a queue for each key head, since windows differ in cost: even ranges of
// windows, passing by those of other classes, took 522 us where this takes 430. Which warp takes a piece, and
// where it stands in the list, changes no value.
constexpr int kPiece = 64;
constexpr int kClasses = 3;
__host__ __device__ constexpr int class_of(int nb) { return nb == 4 ? 0 : nb == 8 ? 1 : 2; }

__global__ void __launch_bounds__(256) k_attn_pieces(const __grid_constant__ AttnParams p) {
    const int w = blockIdx.x * 256 + threadIdx.x, lane = threadIdx.x & 31;
    int cls = -1, pieces = 0;
    if (w < p.windows) {
        const int n = max(attn_offset(p.k_off, p.windows, p.tk, w + 2) - attn_offset(p.k_off, p.windows, p.tk, w + 1), 0);
        const int lq = max(attn_offset(p.q_off, p.windows, p.tq, w + 2) - attn_offset(p.q_off, p.windows, p.tq, w + 1), 0);
        if (n <= p.tiny_max) cls = n <= 32 ? 0 : n <= 64 ? 1 : 2;
        pieces = (lq + kPiece - 1) / kPiece;
    }
#pragma unroll
    for (int c = 0; c < kClasses; ++c) {
        const int mine = cls == c ? pieces : 0;
        int upto = mine;
#pragma unroll
        for (int x = 1; x < 32; x <<= 1) {
            const int v = __shfl_up_sync(0xffffffffu, upto, x);
            if (lane >= x) upto += v;
        }
        int at = 0;
        if (lane == 31 && upto > 0) at = atomicAdd(p.flags + c, upto);
        at = __shfl_sync(0xffffffffu, at, 31) + upto - mine;
        int2* list = reinterpret_cast<int2*>(p.tiny_list) + static_cast<int64_t>(c) * p.tiny_pieces;
        for (int i = 0; i < mine; ++i)
            if (at + i < p.tiny_pieces) list[at + i] = make_int2(w, i * kPiece);
    }
}

// Windows of up to 32 keys (NB = 4), of 33 to 64 (NB = 8) or of 65 to 128 (NB = 16): apart, so that the few
// keys' registers let more warps hide each other's latency, which bounds this kernel.
template <typename T, int DB, int NB, bool BIAS>
__global__ void __launch_bounds__(32 * kWarps, tiny_fwd_blocks(DB, NB)) k_attn_fwd_tiny(const __grid_constant__ AttnParams p) {
    extern __shared__ __align__(16) unsigned char smem_raw[];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int group = p.heads / p.kv_heads, entries = BIAS ? bias_entries(p.bias) : 0;
    const int listed = min(p.flags[class_of(NB)], p.tiny_pieces);
    if (listed == 0) return;
    const Share sh = share_of(p.kv_heads);
    const int side = p.kv_heads >= 4 ? 4 : p.kv_heads >= 2 ? 2 : 1;
    TinyPos<NB>* kp = reinterpret_cast<TinyPos<NB>*>(smem_raw) + warp;
    float* E = reinterpret_cast<float*>(smem_raw + sizeof(TinyPos<NB>) * kWarps);
    if constexpr (BIAS) {
        for (int e = threadIdx.x; e < side * group * entries; e += 32 * kWarps) {
            const int head = blockIdx.y * side * group + e / entries;
            E[e] = head < p.heads ? bias_entry(p.bias, p.heads, head, e % entries) : 0.0f;
        }
        __syncthreads();
    }
    if (sh.kvh >= p.kv_heads) return;
    const float* Eh = E + (sh.kvh % side) * group * entries;
    const int2* list = reinterpret_cast<const int2*>(p.tiny_list) + static_cast<int64_t>(class_of(NB)) * p.tiny_pieces;
    int* queue = p.flags + kClasses + class_of(NB) * p.kv_heads + sh.kvh;
    int item = 0;
    if (lane == 0) item = atomicAdd(queue, 1);
    for (;;) {
        const int now = __shfl_sync(0xffffffffu, item, 0);
        if (now >= listed) break;
        if (lane == 0) item = atomicAdd(queue, 1);  // the next one, known by the time it is wanted
        const int2 piece = list[now];
        const int w = piece.x;
        const int q0 = attn_offset(p.q_off, p.windows, p.tq, w + 1), lq = max(attn_offset(p.q_off, p.windows, p.tq, w + 2) - q0, 0);
        const int k0 = attn_offset(p.k_off, p.windows, p.tk, w + 1), n = max(attn_offset(p.k_off, p.windows, p.tk, w + 2) - k0, 0);
        const int r_begin = piece.y, r_end = min(r_begin + kPiece, lq);
        if (n == 0) {  // nothing to see: zeros
            for (int r = r_begin * group + lane; r < r_end * group; r += 32) {
                const int64_t token = q0 + r / group, head = sh.kvh * group + r % group;
                T* out = static_cast<T*>(p.out) + (token * p.heads + head) * p.dim;
                for (int c = 0; c < p.dim; ++c) out[c] = from_f<T>(0.0f);
                if (p.lse != nullptr) p.lse[head * p.tq + token] = INFINITY;
            }
            continue;
        }
        if constexpr (NB >= 8) {
            tiny_forward<T, DB, NB, BIAS>(p, sh.kvh, group, q0, lq, k0, n, r_begin, r_end, kp, Eh, entries);
        } else {
            if (n <= 16)
                tiny_forward<T, DB, 2, BIAS>(p, sh.kvh, group, q0, lq, k0, n, r_begin, r_end, reinterpret_cast<TinyPos<2>*>(kp), Eh, entries);
            else
                tiny_forward<T, DB, NB, BIAS>(p, sh.kvh, group, q0, lq, k0, n, r_begin, r_end, kp, Eh, entries);
        }
    }
}

// ---- backward -------------------------------------------------------------------------------
// 32 columns and 32 keys at most: dk and dv of the window stay in registers. Windows of up to 16 keys
// (NB = 2) and of 17 to 32 (NB = 4) apart, as in the forward. The bias gradient
// goes into the warp's own 32-bit integers, at a scale of each head's that leaves room for what was added
// since they were last moved to its fp64 sums. A step of 16 rows stands at 2^20 at least: a scale kept from
// a window, or a head, of larger gradients would round the smaller ones away (entries that only these
// reach lost 24% at 2^-16 of the larger ones).
// A warp's sums of the bias gradient.
struct TinySums {
    double* acc;   // [group][n]
    int* I;        // [group][n], times the head's `fixed`
    float* state;  // [group][2], `fixed` and `used` of the heads that are not worked on
    int n;         // entries; 0: no gradient is wanted
    int head;      // of the group
    float fixed, used;
    __device__ __forceinline__ void enter(int head_) {
        head = head_;
        fixed = state[2 * head];
        used = state[2 * head + 1];
    }
    __device__ __forceinline__ void leave() {
        __syncwarp();
        if ((threadIdx.x & 31) == 0) state[2 * head] = fixed, state[2 * head + 1] = used;
        __syncwarp();
    }
    // the head's integers to the fp64 sums
    __device__ __forceinline__ void flush() {
        __syncwarp();
        const double unit = fixed > 0.0f ? 1.0 / static_cast<double>(fixed) : 0.0;
        for (int e = head * n + (threadIdx.x & 31); e < (head + 1) * n; e += 32) {
            const int v = I[e];
            if (v != 0) acc[e] += static_cast<double>(v) * unit, I[e] = 0;
        }
        __syncwarp();
        used = 0.0f;
    }
    // Room for terms of this size altogether, in up to 512 roundings of half a step.
    __device__ __forceinline__ void reserve(float size) {
        if (size > 0.0f && !(size * fixed >= 1048576.0f && used + size * fixed + 512.0f < 1073741824.0f)) {
            const float to = exp2f(static_cast<float>(min(max(23 - ilogbf(size), -126), 126)));
            if (to != fixed || used + size * fixed + 512.0f >= 1073741824.0f) {
                flush();
                fixed = to;
            }
        }
        used += size * fixed + 512.0f;
    }
};

// One window and key head, rows [r_begin, r_end), with NK blocks of 8 keys.
template <typename T, int NK, bool BIAS>
__device__ __forceinline__ void tiny_backward(const AttnParams& p, int kvh, int group, int q0, int lq, int k0, int n, int r_begin, int r_end,
                                              TinyPos<NK < 2 ? 2 : NK>* kp, const float* E, int entries, float up, TinySums& ts) {
    constexpr int NP = NK < 2 ? 2 : NK;  // blocks of positions
    constexpr int NM = (NK + 1) / 2;     // 16-key steps
    const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const float c2 = p.scale * kLog2e;
    uint32_t kr[NK][1][4], vr[NK][1][4], kt[NK][4];
    float dk[NM][1][4][4] = {}, dv[NM][1][4][4] = {};
    {
        const Rows<T, 1> rk(p.k, p.k_st, p.k_sh, p.dim, kvh), rv(p.v, p.v_st, p.v_sh, p.dim, kvh);
#pragma unroll
        for (int kb = 0; kb < NK; ++kb) {
            rk.load(kr[kb], k0 + 8 * kb + g, 8 * kb + g < n);
            rv.load(vr[kb], k0 + 8 * kb + g, 8 * kb + g < n);
        }
#pragma unroll
        for (int kb = 0; kb < NK; ++kb)
#pragma unroll
            for (int j = 0; j < 4; ++j) kt[kb][j] = transpose8(kr[kb][0][j]);
    }
    Range krange{0, 0, 0, 0};
    if (BIAS) krange = tiny_key_pos<NP>(kp, p.bias, k0, n);
    const int left = n - 2 * t;  // key 8 kb + 2 t + i is there where 8 kb + i < left
    for (int gh = 0; gh < group; ++gh) {
        const int head = kvh * group + gh;
        if (BIAS && ts.n > 0) ts.enter(gh);
        const Rows<T, 1> rq(p.q, p.q_st, p.q_sh, p.dim, head), rg(p.dout, p.do_st, p.do_sh, p.dim, head);
        const float* Eh = E + gh * entries;
        // of row g: the next rows to load, and the rows to write
        const T* from_q = rq.p + static_cast<int64_t>(q0 + r_begin + g) * p.q_st;
        const T* from_g = rg.p + static_cast<int64_t>(q0 + r_begin + g) * p.do_st;
        const float* lse_at = p.lse + static_cast<int64_t>(head) * p.tq + q0 + r_begin + g;
        T* to = static_cast<T*>(p.dq) + (static_cast<int64_t>(q0 + r_begin + g) * p.heads + head) * p.dim;
        const int64_t to_step = static_cast<int64_t>(8) * p.heads * p.dim;
        uint32_t nqa[1][4], nqb[1][4], nga[1][4], ngb[1][4];
        float nl[2];
        auto fetch = [&](int r0) {
            const bool a = r0 + g < r_end, b = r0 + 8 + g < r_end;
            rq.load_at(nqa, from_q, a);
            rq.load_at(nqb, from_q + 8 * p.q_st, b);
            rg.load_at(nga, from_g, a);
            rg.load_at(ngb, from_g + 8 * p.do_st, b);
            nl[0] = a ? __ldg(lse_at) : INFINITY;
            nl[1] = b ? __ldg(lse_at + 8) : INFINITY;
            from_q += 16 * p.q_st;
            from_g += 16 * p.do_st;
            lse_at += 16;
        };
        fetch(r_begin);
        for (int r0 = r_begin; r0 < r_end; r0 += 16, to += 2 * to_step) {
            uint32_t qa[4], qb[4], ga[4], gb[4];
            const float lse[2] = {nl[0], nl[1]};
#pragma unroll
            for (int j = 0; j < 4; ++j) qa[j] = nqa[0][j], qb[j] = nqb[0][j], ga[j] = nga[0][j], gb[j] = ngb[0][j];
            fetch(r0 + 16);
            float s[NK][4], dp[NK][4];
#pragma unroll
            for (int kb = 0; kb < NK; ++kb) {
#pragma unroll
                for (int i = 0; i < 4; ++i) s[kb][i] = dp[kb][i] = 0.0f;
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    mma16<T>(s[kb], qa[2 * h], qb[2 * h], qa[2 * h + 1], qb[2 * h + 1], kr[kb][0][2 * h], kr[kb][0][2 * h + 1]);
                    mma16<T>(dp[kb], ga[2 * h], gb[2 * h], ga[2 * h + 1], gb[2 * h + 1], vr[kb][0][2 * h], vr[kb][0][2 * h + 1]);
                }
            }
            const TinyBias<NP> tb(p.bias, kp, krange, q0, lq - 1, BIAS ? r0 : 0, BIAS);
            int at[BIAS ? NK : 1][4];  // entries of the map
            if constexpr (BIAS) {
                if (tb.linear) {
#pragma unroll
                    for (int kb = 0; kb < NK; ++kb)
#pragma unroll
                        for (int i = 0; i < 4; ++i) at[kb][i] = tb.entry_linear(i >> 1, kb, i & 1);
                } else {
#pragma unroll
                    for (int kb = 0; kb < NK; ++kb)
#pragma unroll
                        for (int i = 0; i < 4; ++i) at[kb][i] = tb.entry(i >> 1, kb, i & 1);
                }
            }
            float delta[2] = {0.0f, 0.0f};
#pragma unroll
            for (int kb = 0; kb < NK; ++kb)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float x = BIAS ? fmaf(s[kb][i], c2, Eh[at[kb][i]]) - lse[i >> 1] : fmaf(s[kb][i], c2, -lse[i >> 1]);
                    s[kb][i] = 8 * kb + (i & 1) < left ? ex2(x) : 0.0f;
                }
            if (__any_sync(0xffffffffu, is_far(lse[0]) || is_far(lse[1]))) {
                const int64_t row = static_cast<int64_t>(head) * p.tq + q0 + r0 + g;
                const float f[2] = {far_factor(p, row, lse[0]), far_factor(p, row + 8, lse[1])};
#pragma unroll
                for (int kb = 0; kb < NK; ++kb)
#pragma unroll
                    for (int i = 0; i < 4; ++i) s[kb][i] *= f[i >> 1];
            }
#pragma unroll
            for (int kb = 0; kb < NK; ++kb)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const bool on = 8 * kb + (i & 1) < left;
                    dp[kb][i] = on ? dp[kb][i] : 0.0f;
                    delta[i >> 1] = fmaf(s[kb][i], dp[kb][i], delta[i >> 1]);
                }
            delta[0] = quad_sum(delta[0]);
            delta[1] = quad_sum(delta[1]);
            uint32_t pp[2 * NM][2], pd[2 * NM][2];
            if (NK == 1) pp[1][0] = pp[1][1] = pd[1][0] = pd[1][1] = 0u;
            float size = 0.0f;
#pragma unroll
            for (int kb = 0; kb < NK; ++kb) {
                pp[kb][0] = pack2(s[kb][0], s[kb][1], T{});
                pp[kb][1] = pack2(s[kb][2], s[kb][3], T{});
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    dp[kb][i] = s[kb][i] * (dp[kb][i] - delta[i >> 1]);
                    if (BIAS) size += fabsf(dp[kb][i]);
                }
                pd[kb][0] = pack2(dp[kb][0] * up, dp[kb][1] * up, T{});
                pd[kb][1] = pack2(dp[kb][2] * up, dp[kb][3] * up, T{});
            }
            float dq[1][4][4] = {};
#pragma unroll
            for (int kk = 0; kk < NM; ++kk)
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    mma16<T>(dq[0][j], pd[2 * kk][0], pd[2 * kk][1], pd[2 * kk + 1][0], pd[2 * kk + 1][1], kt[2 * kk][j],
                             NK == 1 ? 0u : kt[NK == 1 ? 0 : 2 * kk + 1][j]);
#pragma unroll
            for (int j = 0; j < 4; ++j) qa[j] = transpose8(qa[j]), qb[j] = transpose8(qb[j]), ga[j] = transpose8(ga[j]), gb[j] = transpose8(gb[j]);
#pragma unroll
            for (int m = 0; m < NM; ++m) {
                const uint32_t a0 = transpose8(pp[2 * m][0]), a1 = NK == 1 ? 0u : transpose8(pp[2 * m + 1][0]),
                               a2 = transpose8(pp[2 * m][1]), a3 = NK == 1 ? 0u : transpose8(pp[2 * m + 1][1]);
                const uint32_t d0 = transpose8(pd[2 * m][0]), d1 = NK == 1 ? 0u : transpose8(pd[2 * m + 1][0]),
                               d2 = transpose8(pd[2 * m][1]), d3 = NK == 1 ? 0u : transpose8(pd[2 * m + 1][1]);
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    mma16<T>(dv[m][0][j], a0, a1, a2, a3, ga[j], gb[j]);
                    mma16<T>(dk[m][0][j], d0, d1, d2, d3, qa[j], qb[j]);
                }
            }
            if constexpr (BIAS) {
                if (ts.n > 0) {
                    size = warp_sum(size);
                    const bool bad = !is_finite(size);
                    if (bad) {
                        size = 0.0f;
#pragma unroll
                        for (int kb = 0; kb < NK; ++kb)
#pragma unroll
                            for (int i = 0; i < 4; ++i)
                                if (is_finite(dp[kb][i])) size += fabsf(dp[kb][i]);
                        size = fminf(warp_sum(size), 3.0e38f);
                    }
                    ts.reserve(size);
                    int* I = ts.I + gh * entries;
#pragma unroll
                    for (int kb = 0; kb < NK; ++kb)
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const float x = dp[kb][i];
                            if (bad && !is_finite(x))
                                bias_mark_bad(p, head, at[kb][i]);
                            else if (x != 0.0f)
                                atomicAdd(I + at[kb][i], __float2int_rn(x * ts.fixed));
                        }
                }
            }
            if (r0 + g < r_end) store_row16<T, 1>(to, p.dim, dq, 0, p.scale / up);
            if (r0 + g + 8 < r_end) store_row16<T, 1>(to + to_step, p.dim, dq, 1, p.scale / up);
        }
        if (BIAS && ts.n > 0) ts.leave();
    }
#pragma unroll
    for (int m = 0; m < NM; ++m)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int j = 16 * m + 8 * h + g;
            if (j >= n) continue;
            const int64_t at = (static_cast<int64_t>(k0 + j) * p.kv_heads + kvh) * p.dim;
            if (p.qsplits == 1) {
                store_row16<T, 1>(static_cast<T*>(p.dk) + at, p.dim, dk[m], h, p.scale / up);
                store_row16<T, 1>(static_cast<T*>(p.dv) + at, p.dim, dv[m], h, 1.0f);
            } else {
                const int64_t part = static_cast<int64_t>(blockIdx.z) * p.tk * p.kv_heads * p.dim + at;
#pragma unroll
                for (int b = 0; b < 4; ++b)
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        const int c = 8 * t + 2 * b + i;
                        if (c >= p.dim) continue;
                        p.part_dk[part + c] = dk[m][0][b][2 * h + i] * (p.scale / up);
                        p.part_dv[part + c] = dv[m][0][b][2 * h + i];
                    }
            }
        }
}

template <typename T, int NB, bool BIAS>
__global__ void __launch_bounds__(32 * kWarps, tiny_bwd_blocks(NB)) k_attn_bwd_tiny(const __grid_constant__ AttnParams p, int first_part) {
    extern __shared__ __align__(16) unsigned char smem_raw[];
    const int warp = threadIdx.x >> 5;
    const int group = p.heads / p.kv_heads, entries = BIAS ? bias_entries(p.bias) : 0;
    const bool grad_bias = BIAS && p.bias_part != nullptr;
    const Share sh = share_of(p.kv_heads);
    const int side = p.kv_heads >= 4 ? 4 : p.kv_heads >= 2 ? 2 : 1;
    TinyPos<NB>* kp = reinterpret_cast<TinyPos<NB>*>(smem_raw) + warp;
    double* acc_all = reinterpret_cast<double*>(smem_raw + sizeof(TinyPos<NB>) * kWarps);
    int* I_all = reinterpret_cast<int*>(acc_all + (grad_bias ? kWarps * group * entries : 0));
    float* E = reinterpret_cast<float*>(I_all + (grad_bias ? kWarps * group * entries : 0));
    float* state = E + side * group * entries;  // of the warps' sums
    if constexpr (BIAS) {
        for (int e = threadIdx.x; e < side * group * entries; e += 32 * kWarps) {
            const int head = blockIdx.y * side * group + e / entries;
            E[e] = head < p.heads ? bias_entry(p.bias, p.heads, head, e % entries) : 0.0f;
        }
        if (grad_bias)
            for (int e = threadIdx.x; e < kWarps * group * entries; e += 32 * kWarps) acc_all[e] = 0.0, I_all[e] = 0;
        if (grad_bias)
            for (int e = threadIdx.x; e < kWarps * group * 2; e += 32 * kWarps) state[e] = 0.0f;
        __syncthreads();
    }
    const bool mine = sh.kvh < p.kv_heads;
    const int kvh = mine ? sh.kvh : 0;
    const float* Eh = E + (kvh % side) * group * entries;
    TinySums ts{acc_all + warp * group * entries, I_all + warp * group * entries, state + warp * group * 2, grad_bias ? entries : 0, 0, 0.0f, 0.0f};

    // the windows of this kernel's class, as listed
    const int* list = p.tiny_list + (NB == 4 ? p.windows : 0);
    const int listed = p.flags[NB == 4 ? 2 : 1];
    for (int item = mine ? sh.first : listed; item < listed; item += sh.step) {
        const int w = list[item];
        const float up = ds_scale<T>(p, w, kvh);
        const int q0 = attn_offset(p.q_off, p.windows, p.tq, w + 1), lq = max(attn_offset(p.q_off, p.windows, p.tq, w + 2) - q0, 0);
        const int k0 = attn_offset(p.k_off, p.windows, p.tk, w + 1), n = max(attn_offset(p.k_off, p.windows, p.tk, w + 2) - k0, 0);
        const int per = ((lq + 15) / 16 + p.qsplits - 1) / p.qsplits * 16;
        const int r_begin = min(static_cast<int>(blockIdx.z) * per, lq), r_end = min(r_begin + per, lq);
        if constexpr (NB == 4) {
            tiny_backward<T, 4, BIAS>(p, kvh, group, q0, lq, k0, n, r_begin, r_end, kp, Eh, entries, up, ts);
        } else {
            if (n <= 8)
                tiny_backward<T, 1, BIAS>(p, kvh, group, q0, lq, k0, n, r_begin, r_end, kp, Eh, entries, up, ts);
            else
                tiny_backward<T, 2, BIAS>(p, kvh, group, q0, lq, k0, n, r_begin, r_end, kp, Eh, entries, up, ts);
        }
    }
    if constexpr (BIAS)
        if (grad_bias) {
            for (int gh = 0; gh < group; ++gh) {
                ts.enter(gh);
                ts.flush();
            }
            // the warps of one key head, in order, make one part
            __syncthreads();
            for (int e = threadIdx.x; e < side * group * entries; e += 32 * kWarps) {
                const int s = e / (group * entries), head = (blockIdx.y * side + s) * group + e / entries % group;
                if (head >= p.heads) continue;
                double sum = 0.0;
                for (int v = s; v < kWarps; v += side) sum += acc_all[v * group * entries + e % (group * entries)];
                p.bias_part[(static_cast<int64_t>(head) * p.bias_parts + first_part + blockIdx.z * gridDim.x + blockIdx.x) * entries + e % entries] = sum;
            }
        }
}

}  // namespace

// Blocks for each set of key heads: resident ones, or as many as the windows fill.
static int tiny_blocks(const AttnParams& p, int resident, int z) {
    const int side = p.kv_heads >= 4 ? 4 : p.kv_heads >= 2 ? 2 : 1, sets = (p.kv_heads + side - 1) / side;
    const int per = (resident * 148 + sets * z - 1) / (sets * z), most = (p.windows + kWarps / side - 1) / (kWarps / side);
    return most < 1 ? 1 : most < per ? most : per;
}
int attn_tiny_pieces(int tq, int windows) { return tq / kPiece + windows; }
int attn_tiny_forward_counters(int kv_heads) { return kClasses * (1 + kv_heads); }
int attn_tiny_lists() { return kClasses; }
int attn_tiny_backward_blocks(const AttnParams& p) { return tiny_blocks(p, 2, p.qsplits); }  // of each of the two kernels

namespace {
int sets_of(const AttnParams& p) {
    const int side = p.kv_heads >= 4 ? 4 : p.kv_heads >= 2 ? 2 : 1;
    return (p.kv_heads + side - 1) / side;
}
int heads_of_block(const AttnParams& p) {
    return (p.kv_heads >= 4 ? 4 : p.kv_heads >= 2 ? 2 : 1) * (p.heads / p.kv_heads);
}

template <typename T, int DB, int NB, bool BIAS>
cudaError_t fwd_one(const AttnParams& p, cudaStream_t s) {
    const int bytes = BIAS ? static_cast<int>(sizeof(TinyPos<NB>)) * kWarps + 4 * heads_of_block(p) * bias_entries(p.bias) : 0;
    cudaError_t err = allow_smem(k_attn_fwd_tiny<T, DB, NB, BIAS>);
    if (err != cudaSuccess) return err;
    // as many blocks as stay resident, or as there can be pieces
    const int side = p.kv_heads >= 4 ? 4 : p.kv_heads >= 2 ? 2 : 1, sets = sets_of(p);
    const int per = (148 * tiny_fwd_blocks(DB, NB) + sets - 1) / sets, most = (p.tiny_pieces + kWarps / side - 1) / (kWarps / side);
    k_attn_fwd_tiny<T, DB, NB, BIAS><<<dim3(most < per ? most : per, sets), 32 * kWarps, bytes, s>>>(p);
    return cudaGetLastError();
}
template <typename T, int NB, bool BIAS>
cudaError_t bwd_one(const AttnParams& p, int first_part, cudaStream_t s) {
    const int64_t entries = BIAS ? bias_entries(p.bias) : 0, group = p.heads / p.kv_heads;
    const int bytes = static_cast<int>(sizeof(TinyPos<NB>) * kWarps + 4 * heads_of_block(p) * entries +
                                       (p.bias_part != nullptr ? kWarps * group * (12 * entries + 8) : 0));
    cudaError_t err = allow_smem(k_attn_bwd_tiny<T, NB, BIAS>);
    if (err != cudaSuccess) return err;
    k_attn_bwd_tiny<T, NB, BIAS><<<dim3(p.tiny_blocks, sets_of(p), p.qsplits), 32 * kWarps, bytes, s>>>(p, first_part);
    return cudaGetLastError();
}
template <typename T, bool BIAS>
cudaError_t fwd_bias(const AttnParams& p, cudaStream_t s) {
    if (p.dim > 32) return fwd_one<T, 2, 4, BIAS>(p, s);
    cudaError_t err = fwd_one<T, 1, 16, BIAS>(p, s);
    if (err == cudaSuccess) err = fwd_one<T, 1, 8, BIAS>(p, s);
    return err != cudaSuccess ? err : fwd_one<T, 1, 4, BIAS>(p, s);
}
template <typename T, bool BIAS>
cudaError_t bwd_bias(const AttnParams& p, cudaStream_t s) {
    const cudaError_t err = bwd_one<T, 4, BIAS>(p, 0, s);
    return err != cudaSuccess ? err : bwd_one<T, 2, BIAS>(p, p.tiny_blocks * p.qsplits, s);
}
template <typename T>
cudaError_t fwd_type(const AttnParams& p, cudaStream_t s) {
    return p.bias.table != nullptr ? fwd_bias<T, true>(p, s) : fwd_bias<T, false>(p, s);
}
template <typename T>
cudaError_t bwd_type(const AttnParams& p, cudaStream_t s) {
    return p.bias.table != nullptr ? bwd_bias<T, true>(p, s) : bwd_bias<T, false>(p, s);
}

}  // namespace

cudaError_t launch_attn_forward_tiny(const AttnParams& p, int type, cudaStream_t s) {
    cudaError_t err = cudaMemsetAsync(p.flags, 0, sizeof(int) * kClasses * (1 + p.kv_heads), s);
    if (err != cudaSuccess) return err;
    k_attn_pieces<<<(p.windows + 255) / 256, 256, 0, s>>>(p);
    if ((err = cudaGetLastError()) != cudaSuccess) return err;
    return type == kBF16 ? fwd_type<__nv_bfloat16>(p, s) : fwd_type<__half>(p, s);
}
cudaError_t launch_attn_backward_tiny(const AttnParams& p, int type, cudaStream_t s) {
    return type == kBF16 ? bwd_type<__nv_bfloat16>(p, s) : bwd_type<__half>(p, s);
}

}  // namespace oss
