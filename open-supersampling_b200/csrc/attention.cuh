// Window attention over packed windows: the parameters, the walk over the
// windows' tiles and the bucketed position bias that all its kernels share.
//
// Window w holds queries [q_off[w], q_off[w+1]) and keys [k_off[w], k_off[w+1]).
//   s_ij = scale q_i.k_j + table[bucket[clamp(kpos_j - qpos_i)], h]
//   p_ij = softmax over the visible j of s_ij,   o_i = sum_j p_ij v_j
// All softmax arithmetic is in base 2: the kernels hold s log2(e).
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

namespace oss {

constexpr float kLog2e = 1.4426950408889634f;
// Entries of the expanded position bias, (2 ry + 1) (2 rx + 1): a head's bias, its integer gradient sums and
// (in fp32 only where they fit) their fp64 sums stay in shared memory beside the tiles (16 + 16 + 32 KB; fp32 16 + 32 + 32).
constexpr int kMaxBiasEntries = 4096;
constexpr int kMaxHeadDim = 128;
// Positions are clamped to this magnitude on load, so that their differences stay within int32. Linear
// codes count y from a key of the tile: (y - y0) (2 rx + 1) + x, which stays there too where no pair needs clamping.
constexpr int kMaxPosition = 1 << 29;

enum AttnType { kF32 = 0, kBF16 = 1, kF16 = 2 };

struct AttnBias {
    const void* table;       // [buckets][heads], null: no bias
    int table_type;          // AttnType
    int buckets;             // rows of table
    const int32_t* map;      // [2 ry + 1][2 rx + 1] -> row of table; outside [0, buckets): no bias
    int ry, rx;
    const int32_t* q_pos;    // [tq][axes], (y, x) or (x)
    const int32_t* k_pos;    // [tk][axes]
    int axes;
};

struct AttnParams {
    const void *q, *k, *v;
    int64_t q_st, q_sh, k_st, k_sh, v_st, v_sh;  // strides in elements: token, head
    const int32_t *q_off, *k_off;                // [windows + 1]
    int windows, tq, tk;
    int heads, kv_heads, dim;
    float scale;
    int causal;
    AttnBias bias;
    void* out;        // [tq][heads][dim]
    float* lse;       // [heads][tq], base 2, +inf for a row that sees no key; may be null
    float* lse_rest;  // [heads][tq], what rounding took from lse where that is far from 0; may be null
    // What rounding took from out, [tq][heads][dim] of the same type, of windows with more keys than short_max (others'
    // may stay unwritten): dout . out is then right to fp32. With out alone the gradients of long windows were
    // off by half as much again as rounding them makes them, and the bias table's by twice. May be null; 16-bit types.
    void* out_lo;
    int tiny_max;     // windows of up to so many keys (backward: of 1 to so many) go to the warp-level kernels
                      // (attention_tiny.cu); 0: none
    // forward only
    int pack;         // query heads of one key head that share a tile's rows (1 or the group)
    int splits;       // parts that a window's keys are cut into
    float* part_o;    // [splits][tq][heads][dim], splits > 1 only
    float* part_ml;   // [splits][tq][heads][2]
    // backward only
    const void* dout;  // [tq][heads][dim]
    int64_t do_st, do_sh;
    float* delta;        // [heads][tq], sum_j p_ij dp_ij
    void *dq, *dk, *dv;  // contiguous [tq][heads][dim], [tk][kv_heads][dim]
    unsigned long long* bias_acc;  // [buckets][heads], fixed point; zero at the start, as the next two
    unsigned long long* bias_top;  // [buckets][heads], largest magnitude of its entries' sums (bits of a double)
    uint32_t* bias_bad;            // [buckets][heads], nonzero where a term was not finite
    uint32_t* win_max;             // fp16: [windows][kv_heads][2], largest finite |dout| and |v| of a window (bits of an
                                   // fp16 value); zero at the start
    double* bias_part;           // [heads][bias_parts][entries]; null: no gradient of the table
    int bias_tiny, bias_short, bias_parts;  // parts of the tiny and the short windows' blocks, and all of them
    int dq_blocks;               // blocks of the kernel for dq for each head
    // backward of 16-bit types only
    int short_max;      // windows of up to so many keys go to the kernel for short windows
    int qsplits;        // parts that the queries of a tile of keys are cut into
    int tiny_blocks, short_blocks, dkv_blocks;  // blocks of the kernels for each (set of) head(s)
    // flags and tiny_list serve the forward of the few-keys kernels too: counters and queues, and pieces by class
    int* flags;         // [0]: kSomeLong, kSomeShort; [1], [2]: windows of up to 16 and of 17 to 32 keys
    int* tiny_list;     // [2][windows]: those windows, in order
    int tiny_pieces;    // forward: most pieces of a class
    float *part_dk, *part_dv;    // [qsplits][tk][kv_heads][dim], qsplits > 1 only
};

constexpr int kSomeLong = 1;   // a window with more than short_max keys
constexpr int kSomeShort = 2;  // one with more than tiny_max, up to short_max

__host__ __device__ __forceinline__ int bias_entries(const AttnBias& b) {
    return b.table == nullptr ? 0 : (2 * b.ry + 1) * (2 * b.rx + 1);
}

// ---------------------------------------------------------------------------
// Tiles of packed windows without a host read of the offsets.  Window w of the
// W + 2 below (the rows before the first offset and behind the last one are
// windows without partners, so that their outputs are written too) owns the
// slots from floor(off[w] / rows) + w on: that is at least ceil(len / rows) of
// them, the total floor(t / rows) + W + 2 is known on the host, and a slot's
// window is found with a 32-way search (three probes for 32k windows).  Slots
// that come out empty return at once.
__host__ __device__ __forceinline__ int attn_slots(int64_t t, int windows, int rows) {
    return static_cast<int>(t / rows) + windows + 2;
}

__device__ __forceinline__ int attn_offset(const int32_t* off, int windows, int t, int w) {
    if (w <= 0) return 0;
    if (w >= windows + 2) return t;
    return min(max(__ldg(off + w - 1), 0), t);
}

struct AttnTile {
    int window;      // in [0, windows), or -1: rows outside every window
    int begin, len;  // the window's tokens on the walked side
    int first;       // first row of the tile, counted in rows of the window
    int obegin, olen;  // the window's tokens on the other side
};

// Called by whole warps. `per`: rows for each token (packed heads). False: nothing to do.
__device__ __forceinline__ bool attn_tile(const int32_t* off, int t, const int32_t* other, int ot, int windows, int per,
                                          int rows, int slot, AttnTile& tile) {
    const int lane = threadIdx.x & 31;
    int lo = 0, hi = windows + 2;
    while (hi - lo > 1) {
        const int step = (hi - lo + 31) >> 5;
        const int w = lo + lane * step;
        bool before = false;
        if (w < hi) before = static_cast<int>(static_cast<int64_t>(attn_offset(off, windows, t, w)) * per / rows) + w <= slot;
        const unsigned hit = __ballot_sync(0xffffffffu, before) | 1u;
        const int n = __ffs(~hit) == 0 ? 32 : __ffs(~hit) - 1;  // leading probes at or before the slot
        lo += (n - 1) * step;
        hi = min(hi, lo + step);
    }
    tile.begin = attn_offset(off, windows, t, lo);
    tile.len = max(attn_offset(off, windows, t, lo + 1) - tile.begin, 0);
    const int64_t first =
        static_cast<int64_t>(slot - (static_cast<int>(static_cast<int64_t>(tile.begin) * per / rows) + lo)) * rows;
    if (first < 0 || first >= static_cast<int64_t>(tile.len) * per) return false;
    tile.first = static_cast<int>(first);
    tile.window = lo >= 1 && lo <= windows ? lo - 1 : -1;
    tile.obegin = tile.olen = 0;
    if (tile.window >= 0) {
        tile.obegin = attn_offset(other, windows, ot, lo);
        tile.olen = max(attn_offset(other, windows, ot, lo + 1) - tile.obegin, 0);
    }
    return true;
}

// The tiles of slots [slot, end) one after the other: a search for the first, then window by
// window (neighbouring offsets share cache lines).
template <int ROWS>
struct AttnWalk {
    const int32_t *off, *other;
    int t, ot, windows, per;
    int skip;  // where not 0: windows with up to so many tokens on the other side are passed by
    int slot, end, w;
    AttnTile tile;

    // Called by whole warps. False: no tile.
    __device__ __forceinline__ bool start(const int32_t* off_, int t_, const int32_t* other_, int ot_, int windows_, int per_,
                                          int slot_, int end_, int skip_ = 0) {
        off = off_, t = t_, other = other_, ot = ot_, windows = windows_, per = per_, slot = slot_, end = end_;
        skip = skip_;
        const int lane = threadIdx.x & 31;
        int lo = 0, hi = windows + 2;
        while (hi - lo > 1) {
            const int step = (hi - lo + 31) >> 5, at = lo + lane * step;
            const unsigned hit = __ballot_sync(0xffffffffu, at < hi && slot_of(at) <= slot) | 1u;
            const int n = hit == 0xffffffffu ? 32 : __ffs(~hit) - 1;  // leading probes at or before the slot
            lo += (n - 1) * step;
            hi = min(hi, lo + step);
        }
        enter(lo);
        return settle();
    }
    __device__ __forceinline__ bool next() {
        ++slot;
        const int64_t first = static_cast<int64_t>(tile.first) + ROWS;
        if (slot >= end || first >= static_cast<int64_t>(tile.len) * per) return settle();
        tile.first = static_cast<int>(first);
        return true;
    }
    __device__ __forceinline__ int slot_of(int at) const {
        return static_cast<int>(static_cast<uint64_t>(attn_offset(off, windows, t, at)) * static_cast<unsigned>(per) / ROWS) + at;
    }
    __device__ __forceinline__ void enter(int at) {
        w = at;
        tile.begin = attn_offset(off, windows, t, w);
        tile.len = max(attn_offset(off, windows, t, w + 1) - tile.begin, 0);
        tile.window = w >= 1 && w <= windows ? w - 1 : -1;
        tile.obegin = tile.olen = 0;
        if (tile.window >= 0) {
            tile.obegin = attn_offset(other, windows, ot, w);
            tile.olen = max(attn_offset(other, windows, ot, w + 1) - tile.obegin, 0);
        }
    }
    __device__ __forceinline__ bool settle() {
        while (slot < end) {
            const int64_t first = static_cast<int64_t>(slot - slot_of(w)) * ROWS;
            if (first >= 0 && first < static_cast<int64_t>(tile.len) * per && (tile.olen > skip || (tile.olen == 0 && (skip == 0 || tile.window < 0)))) {
                tile.first = static_cast<int>(first);
                return true;
            }
            // the next window to stop at, 32 at a time
            const int lane = threadIdx.x & 31;
            int at = w + 1;
            for (;; at += 32) {
                const int c = at + lane;
                bool stop = c > windows + 1 || slot_of(c) >= end;
                if (!stop) {
                    const int n = c >= 1 && c <= windows ? attn_offset(other, windows, ot, c + 1) - attn_offset(other, windows, ot, c) : 0;
                    stop = attn_offset(off, windows, t, c + 1) > attn_offset(off, windows, t, c) &&
                           (n > skip || (n <= 0 && (skip == 0 || c < 1 || c > windows)));
                }
                const unsigned hit = __ballot_sync(0xffffffffu, stop);
                if (hit != 0u) {
                    at += __ffs(hit) - 1;
                    break;
                }
            }
            if (at > windows + 1) return false;
            enter(at);
            slot = max(slot, slot_of(w));
        }
        return false;
    }
};

// ---------------------------------------------------------------------------
template <typename T>
__device__ __forceinline__ float to_f(T x) {
    return static_cast<float>(x);
}
template <typename T>
__device__ __forceinline__ T from_f(float x);
template <>
__device__ __forceinline__ float from_f<float>(float x) {
    return x;
}
template <>
__device__ __forceinline__ __nv_bfloat16 from_f<__nv_bfloat16>(float x) {
    return __float2bfloat16_rn(x);
}
template <>
__device__ __forceinline__ __half from_f<__half>(float x) {
    return __float2half_rn(x);
}

__device__ __forceinline__ float load_typed(const void* p, int type, int64_t i) {
    if (type == kF32) return static_cast<const float*>(p)[i];
    if (type == kBF16) return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
    return __half2float(static_cast<const __half*>(p)[i]);
}
__device__ __forceinline__ void store_typed(void* p, int type, int64_t i, float x) {
    if (type == kF32)
        static_cast<float*>(p)[i] = x;
    else if (type == kBF16)
        static_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(x);
    else
        static_cast<__half*>(p)[i] = __float2half_rn(x);
}

__device__ __forceinline__ bool is_finite(float x) { return (__float_as_uint(x) & 0x7f800000u) != 0x7f800000u; }
__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// ---- the log of a row's sum ------------------------------------------------------
// A row whose every score is far from 0 (a bias of -1e9 on all its keys) loses the log of its sum beside the
// maximum, and its weights in the backward would be too large by that. What rounding takes is kept there, and
// weights are taken times 2^-rest; a closer row loses less than 2^-14.
constexpr float kFar = 1024.0f;
__device__ __forceinline__ bool is_far(float lse) { return fabsf(lse) > kFar && fabsf(lse) < INFINITY; }
__device__ __forceinline__ void store_lse(const AttnParams& p, int64_t at, float m, float l) {
    const float b = log2f(l), lse = l == 0.0f ? INFINITY : m + b;
    p.lse[at] = lse;
    if (p.lse_rest != nullptr && is_far(lse)) {
        const float bb = lse - m;
        p.lse_rest[at] = (m - (lse - bb)) + (b - bb);
    }
}
__device__ __forceinline__ float far_factor(const AttnParams& p, int64_t at, float lse) {
    return p.lse_rest != nullptr && is_far(lse) ? ex2(-p.lse_rest[at]) : 1.0f;
}

// ---- bias ------------------------------------------------------------------
// A head's expanded bias, times log2(e): entry (dy + ry) (2 rx + 1) + dx + rx. A finite value stays finite: the
// lowest value of fp32 or bf16 lowers its keys (all alike where a row has no others), only minus infinity leaves them no weight.
__device__ __forceinline__ float bias_entry(const AttnBias& b, int heads, int head, int e) {
    const int bucket = __ldg(b.map + e);
    if (bucket < 0 || bucket >= b.buckets) return 0.0f;
    const float x = load_typed(b.table, b.table_type, static_cast<int64_t>(bucket) * heads + head);
    constexpr float kMost = 3.4028234663852886e38f;
    return is_finite(x) ? fminf(fmaxf(x * kLog2e, -kMost), kMost) : x;
}
__device__ __forceinline__ int2 bias_pos(const int32_t* pos, int axes, int64_t token) {
    int2 p = axes == 2 ? make_int2(__ldg(pos + token * 2), __ldg(pos + token * 2 + 1)) : make_int2(0, __ldg(pos + token));
    p.x = min(max(p.x, -kMaxPosition), kMaxPosition);
    p.y = min(max(p.y, -kMaxPosition), kMaxPosition);
    return p;  // .x the first axis (y), .y the second (x)
}
__device__ __forceinline__ int bias_index(const AttnBias& b, int2 qp, int2 kp) {
    const int dy = min(max(kp.x - qp.x, -b.ry), b.ry) + b.ry;
    const int dx = min(max(kp.y - qp.y, -b.rx), b.rx) + b.rx;
    return dy * (2 * b.rx + 1) + dx;
}

// Gradient of the bias: a tile's terms join integer sums, which come out the same in any order, at a
// power of two that keeps the tile's sum of magnitudes m below 2^bits. (A scale for the whole call
// let one large value, even of a row that no window holds, take the bits of all others.)
__device__ __forceinline__ float bias_scale(float m, int bits) {
    return m > 0.0f ? exp2f(static_cast<float>(min(max(bits - 1 - ilogbf(fminf(m, 3.0e38f)), -126), 126))) : 0.0f;
}

// 64-bit add into two shared 32-bit words (native integer atomics; the carry goes by hand).
__device__ __forceinline__ void bias_add_shared(uint32_t* lo, uint32_t* hi, int e, long long v) {
    const uint32_t vl = static_cast<uint32_t>(v);
    uint32_t vh = static_cast<uint32_t>(static_cast<unsigned long long>(v) >> 32);
    const uint32_t old = atomicAdd(lo + e, vl);
    vh += (old + vl < old) ? 1u : 0u;
    if (vh != 0u) atomicAdd(hi + e, vh);
}

__device__ __forceinline__ void bias_mark_bad(const AttnParams& p, int head, int e) {
    const int bucket = __ldg(p.bias.map + e);
    if (bucket >= 0 && bucket < p.bias.buckets) p.bias_bad[static_cast<int64_t>(bucket) * p.heads + head] = 1u;
}

// The sum of finite |ds| of a warp's rows, negative where some is not finite.
template <int N>
__device__ __forceinline__ float warp_size(const float (&ds)[N]) {
    float m = 0.0f;
#pragma unroll
    for (int c = 0; c < N; ++c) m += fabsf(ds[c]);
#pragma unroll
    for (int x = 16; x > 0; x >>= 1) m += __shfl_xor_sync(0xffffffffu, m, x);
    if (is_finite(m)) return m;
    m = 0.0f;
#pragma unroll
    for (int c = 0; c < N; ++c)
        if (is_finite(ds[c])) m += fabsf(ds[c]);
#pragma unroll
    for (int x = 16; x > 0; x >>= 1) m += __shfl_xor_sync(0xffffffffu, m, x);
    return -fmaxf(fminf(m, 3.0e38f), 1.0e-38f);
}

// What rounding x to T takes from it.
template <typename T>
__device__ __forceinline__ float lost_by(float x) {
    const float d = x - to_f(from_f<T>(x));
    return is_finite(d) ? d : 0.0f;
}


// ---- launchers -----------------------------------------------------------------
constexpr int kMaxSmem = 227 * 1024;  // of a block
// Lets a kernel take any shared memory there is. The limit is one for all host threads: set to what a call needs,
// it made the launch of another thread fail that came with a larger map in between.
template <typename K>
cudaError_t allow_smem(K kernel) {
    return cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kMaxSmem);
}

// type: AttnType of q, k, v and out.
cudaError_t launch_attn_forward(const AttnParams& p, int type, cudaStream_t s);
// dtable (null: no gradient of the table).
cudaError_t launch_attn_backward(const AttnParams& p, int type, void* dtable, int sms, cudaStream_t s);
// attention_simt.cu: delta of 16-bit types, where some window is long; p.bias_part to dtable.
cudaError_t launch_attn_delta(const AttnParams& p, int type, int sms, cudaStream_t s);
cudaError_t launch_attn_bias_grad(const AttnParams& p, void* dtable, cudaStream_t s);
// attention_mma.cu, attention_mma_bwd.cu: bf16 and fp16, the forward without the join of split keys.
cudaError_t launch_attn_forward_mma(const AttnParams& p, int type, cudaStream_t s);
// Windows of up to p.tiny_max keys (backward: of 1 to 32), not causal, dim <= 64 (backward: 32).
cudaError_t launch_attn_forward_tiny(const AttnParams& p, int type, cudaStream_t s);
cudaError_t launch_attn_backward_tiny(const AttnParams& p, int type, cudaStream_t s);
int attn_tiny_backward_blocks(const AttnParams& p);
int attn_tiny_pieces(int tq, int windows);
int attn_tiny_forward_counters(int kv_heads);
int attn_tiny_lists();
cudaError_t launch_attn_backward_mma(const AttnParams& p, int type, void* dtable, int sms, cudaStream_t s);
// Waits of the tensor-core kernels that ran out of their limit since the library was loaded.
cudaError_t attn_timeouts(unsigned int* count);
cudaError_t attn_timeouts_bwd(unsigned int* count);

}  // namespace oss
