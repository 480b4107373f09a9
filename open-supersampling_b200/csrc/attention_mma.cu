// Window attention of 16-bit types on the tensor cores (tcgen05): forward.
//
// A block holds 128 query rows and walks its window's keys KT at a time. Four warps do the softmax
// (thread = row = tensor-memory lane), a fifth moves the keys and values and issues the products:
//   S = Q K^T into tensor memory (both operands from shared memory)
//   each thread reads its row of S, keeps the running maximum and sum in registers, and writes
//   the weights back over S as 16-bit values
//   O += P V, P from tensor memory
// K of the next tile is on its way while the softmax runs, V while S is computed (a tensor copy each;
// 16- or 4-byte copies or plain loads where strides or alignment allow none). Two or three blocks
// share an SM and fill each other's waits. Tiles end at the window's last key rounded up to 16,
// whatever KT is: N of S and K of P V are set by it.
// The running maximum that the weights are taken against moves only when a row exceeds it by
// 2^8: O has to be scaled in tensor memory then, which after the first tiles hardly happens.
// With head dims up to 64 the exponentials (16 a clock and SM) bound long windows: 64-key tiles
// leave room for three blocks. With 128 the products do, and 128-key tiles feed them from shared
// memory at the full rate.
#include <cuda.h>

#include "attention_mma.cuh"
#include "internal.h"

namespace oss {
namespace {

// ---- a row again, where a product met what its mask hides --------------------------------
// 0 times a NaN or an infinity behind the causal mask is NaN. A row that comes out not finite is
// summed once more over the keys it sees (which leaves it not finite if one of those is).
template <typename T>
__device__ __noinline__ void forward_row(const AttnParams& p, int64_t token, int head, const int32_t* k_pos0, int64_t kt0, int k0,
                                         int k1, float m, const float* E, int2 qp, uint32_t stage, float* part, float inv) {
    float o[kMaxHeadDim];
    const int kvh = head / (p.heads / p.kv_heads);
    const T* q = static_cast<const T*>(p.q) + token * p.q_st + head * p.q_sh;
    const T* kb = static_cast<const T*>(p.k) + kvh * p.k_sh;
    const T* vb = static_cast<const T*>(p.v) + kvh * p.v_sh;
    for (int c = 0; c < kMaxHeadDim; ++c) o[c] = 0.0f;
    for (int j = k0; j < k1; ++j) {
        float s = 0.0f;
        for (int c = 0; c < p.dim; ++c) s = fmaf(to_f(q[c]), to_f(kb[(kt0 + j) * p.k_st + c]), s);
        s *= p.scale * kLog2e;
        if (k_pos0 != nullptr) s += E[bias_index(p.bias, qp, bias_pos(k_pos0, p.bias.axes, kt0 + j))];
        const float w = to_f(from_f<T>(ex2(s - m)));
        for (int c = 0; c < p.dim; ++c) o[c] = fmaf(w, to_f(vb[(kt0 + j) * p.v_st + c]), o[c]);
    }
    for (int c = 0; c < ((p.dim + 15) & ~15); c += 16) {
        if (part != nullptr)
            write_part(part, o + c, c, p.dim);
        else
            stage16<T>(stage, threadIdx.x, o + c, c, inv);
    }
}

// ---- forward ---------------------------------------------------------------------------
template <int KT, int DP>
struct FwdSmem {
    static constexpr int kBuf = DP == 64 ? 2 : 1;  // tiles of keys, and of values
    static constexpr int kQ = kRows * DP * 2, kK = KT * DP * 2;
    static constexpr int kTiles = kQ + 2 * kBuf * kK;
    static constexpr int kBytes = kTiles + kBuf * static_cast<int>(sizeof(KeyPos<KT>)) + 128;
};

// Keys or values by tensor copies: the map's axes are (column, head, token) or (column, token, head).
struct TileMaps {
    CUtensorMap k, v;
    int use;          // 0: no maps
    int k_tokens_y, v_tokens_y;  // tokens are the second axis
};

// A tile of rows by one warp, where no tensor copy can do it.
template <typename T>
__device__ __forceinline__ void warp_load(uint32_t dst, int panel_rows, const void* q, int64_t st, int64_t sh, int dim, int head, int64_t token,
                                          int rows, int rows_pad) {
    const Loader<T, 32> l(q, st, sh, dim, head);
    if (!l.on) return;
    for (int r = l.r0; r < rows_pad; r += l.step) {
        const uint32_t to = dst + (l.c >> 3) * panel_rows * 128 + r * 128 + (((l.c & 7) ^ (r & 7)) << 4);
        const T* from = l.p + (token + r) * st;
        if (l.zero || r >= rows)
            Loader<T, 32>::store_zero(to);
        else if (l.vec)
            tc::cp_async16(to, from);
        else
            l.store_some(to, from);
    }
}

template <typename T, int KT, int DP, bool BIAS>
__global__ void __launch_bounds__(kRows + 32, KT == 64 ? 3 : 2) k_attn_fwd_mma(const __grid_constant__ AttnParams p, const __grid_constant__ TileMaps maps) {
    using L = FwdSmem<KT, DP>;
    constexpr int kCols = KT + DP, kBuf = L::kBuf;  // 128 or 256 columns: S (P over it), then O
    constexpr int kBf16 = std::is_same<T, __nv_bfloat16>::value ? 1 : 0;
    extern __shared__ __align__(16) unsigned char smem_raw[];
    unsigned char* base = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    const uint32_t sq = tc::smem_addr(base), sk = sq + L::kQ, sv = sk + kBuf * L::kK;
    KeyPos<KT>* kps = reinterpret_cast<KeyPos<KT>*>(base + L::kTiles);
    uint64_t* bars = reinterpret_cast<uint64_t*>(kps + kBuf);
    uint32_t* slot_tmem = reinterpret_cast<uint32_t*>(bars + 14);
    volatile int* dead = reinterpret_cast<volatile int*>(bars + 15);
    float* E = reinterpret_cast<float*>(bars + 16);
    const uint32_t bar0 = tc::smem_addr(bars);
    // barriers: Q there, S done, P there, O done, then for each buffer K there, V there, positions there, positions read
    const uint32_t bar_q = bar0, bar_s = bar0 + 8, bar_p = bar0 + 16, bar_o = bar0 + 24;
    auto bar_k = [&](int b) { return bar0 + 32 + 8 * b; };
    auto bar_v = [&](int b) { return bar0 + 48 + 8 * b; };
    auto bar_pos = [&](int b) { return bar0 + 64 + 8 * b; };
    auto bar_pos_read = [&](int b) { return bar0 + 80 + 8 * b; };

    const int tid = threadIdx.x, warp = tid >> 5;
    const int head0 = blockIdx.y * p.pack, kvh = head0 / (p.heads / p.kv_heads);
    const int entries = BIAS ? bias_entries(p.bias) : 0, dim16 = (p.dim + 15) & ~15;
    const float c2 = p.scale * kLog2e;

    const int slots = attn_slots(static_cast<int64_t>(p.tq) * p.pack, p.windows, kRows);
    const int chunk = (slots + gridDim.x - 1) / gridDim.x;
    // causal windows: the last tiles see the most keys and go first
    const int slot0 = (p.causal ? gridDim.x - 1 - blockIdx.x : blockIdx.x) * chunk;
    AttnWalk walk;
    bool more = walk.start(p.q_off, p.tq, p.k_off, p.tk, p.windows, p.pack, kRows, slot0, min(slots, slot0 + chunk), p.tiny_max);
    if (!more) return;

    if (tid == 0) {
        for (int b = 0; b < 10; ++b) tc::mbar_init(bar0 + 8 * b, b == 0 || b == 2 ? kRows : 1);
        tc::mbar_init(bar_pos_read(0), kRows);
        tc::mbar_init(bar_pos_read(1), kRows);
        tc::mbar_init_fence();
        *dead = 0;
    }
    if (warp == 0) tc::tmem_alloc<kCols>(tc::smem_addr(slot_tmem));
    if constexpr (BIAS)
        for (int e = tid; e < entries * p.pack; e += kRows + 32) E[e] = bias_entry(p.bias, p.heads, head0 + e / entries, e % entries);
    tc::fence_before();
    __syncthreads();
    tc::fence_after();
    const uint32_t tmem = *slot_tmem;

    // the tiles of keys of a tile of queries
    struct Keys {
        int rows, shift, least, tile0, tile1, most;
    };
    auto keys_of = [&](const AttnTile& t) {
        Keys k;
        k.rows = min(kRows, t.len * p.pack - t.first);
        k.shift = t.olen - t.len;
        k.most = k.least = t.olen;  // keys that the last row sees, and the first
        if (p.causal) {
            k.most = min(max((p.pack > 1 ? (t.first + k.rows - 1) / p.pack : t.first + k.rows - 1) + k.shift + 1, 0), t.olen);
            k.least = min(max((p.pack > 1 ? t.first / p.pack : t.first) + k.shift + 1, 0), t.olen);
        }
        k.tile0 = 0, k.tile1 = (k.most + KT - 1) / KT;
        if (p.splits > 1) {
            const int per = (k.tile1 + p.splits - 1) / p.splits;
            k.tile0 = min(static_cast<int>(blockIdx.z) * per, k.tile1);
            k.tile1 = min(k.tile0 + per, k.tile1);
        }
        return k;
    };

    if (warp == 4) {
        // ---- keys, values and products
        const int lane = tid & 31;
        const uint32_t id_o = tc::idesc(kBf16, dim16, false, true);
        int par_q = 0, par_s = 0, par_p = 0, par_o = 0, count = 0;  // count: tiles of keys so far
        for (; more; more = walk.next()) {
            const AttnTile& t = walk.tile;
            const Keys kk = keys_of(t);
            if (kk.tile0 >= kk.tile1) continue;
            const int before = count - kk.tile0;  // tiles of keys before tile 0 of this one
            auto tile_keys = [&](int kt) { return min(KT, kk.most - kt * KT); };
            auto load = [&](bool values, int kt) {  // tile kt of K or V
                const int b = kBuf == 2 ? (before + kt) & 1 : 0, n = tile_keys(kt);
                const uint32_t dst = (values ? sv : sk) + b * L::kK;
                const int token = t.obegin + kt * KT;
                if (maps.use) {
                    if (tc::elect_one()) {
                        const uint32_t bar = values ? bar_v(b) : bar_k(b);
                        const int panels = dim16 > 64 ? 2 : 1;
                        const bool ty = values ? maps.v_tokens_y : maps.k_tokens_y;
                        tc::mbar_expect(bar, panels * KT * 128);
                        for (int h = 0; h < panels; ++h)
                            tc::tma_load(dst + h * KT * 128, values ? &maps.v : &maps.k, bar, 64 * h, ty ? token : kvh, ty ? kvh : token);
                    }
                } else if (values) {
                    warp_load<T>(dst, KT, p.v, p.v_st, p.v_sh, p.dim, kvh, token, n, (n + 15) & ~15);
                    tc::cp_async_commit();
                } else {
                    warp_load<T>(dst, KT, p.k, p.k_st, p.k_sh, p.dim, kvh, token, n, (n + 15) & ~15);
                    tc::cp_async_commit();
                }
                if (BIAS && !values) {
                    const int parity = ((before + kt) / kBuf) & 1;
                    tc::mbar_wait(bar_pos_read(b), parity ^ 1, dead);  // passes at once the first time
                    load_key_pos_warp<KT>(kps + b, p.bias, token, n);
                    __syncwarp();
                    if (lane == 0) tc::mbar_arrive(bar_pos(b));
                }
            };
            load(false, kk.tile0);
            load(true, kk.tile0);
            if (kBuf == 2 && kk.tile0 + 1 < kk.tile1) load(false, kk.tile0 + 1);
            tc::mbar_wait(bar_q, par_q, dead);
            par_q ^= 1;
            for (int kt = kk.tile0; kt < kk.tile1; ++kt, ++count) {
                const int b = kBuf == 2 ? count & 1 : 0, parity = (count / kBuf) & 1;
                const int n = tile_keys(kt), n16 = (n + 15) & ~15;
                if (kt > kk.tile0) {  // O of the tile before: P and its values are free
                    tc::mbar_wait(bar_o, par_o, dead);
                    par_o ^= 1;
                    if (kBuf == 1) load(true, kt);
                }
                if (maps.use) {
                    tc::mbar_wait(bar_k(b), parity, dead);
                } else {
                    tc::cp_async_wait<0>();
                    tc::fence_async();
                    __syncwarp();
                }
                if (tc::elect_one()) {
                    tc::fence_after();
                    tc::mma_nt<DP, kRows, KT>(tmem, sq, sk + b * L::kK, dim16, tc::idesc(kBf16, n16, false, false));
                    tc::commit(bar_s);
                }
                __syncwarp();
                if (kBuf == 2 && kt + 1 < kk.tile1) {
                    // the other buffers: of values since O above, of keys since the S before
                    load(true, kt + 1);
                }
                tc::mbar_wait(bar_s, par_s, dead);
                par_s ^= 1;
                if (kt + kBuf < kk.tile1) load(false, kt + kBuf);
                tc::mbar_wait(bar_p, par_p, dead);
                par_p ^= 1;
                if (maps.use) {
                    tc::mbar_wait(bar_v(b), parity, dead);
                    if (n < n16) {  // what follows the window's last value meets weights of 0: it must not be NaN
                        const int chunks = dim16 / 8;
                        for (int i = lane; i < (n16 - n) * chunks; i += 32) {
                            const int r = n + i / chunks, c = i % chunks;
                            Loader<T, 32>::store_zero(sv + b * L::kK + (c >> 3) * KT * 128 + r * 128 + (((c & 7) ^ (r & 7)) << 4));
                        }
                        tc::fence_async();
                        __syncwarp();
                    }
                } else {
                    tc::cp_async_wait<0>();
                    tc::fence_async();
                    __syncwarp();
                }
                if (tc::elect_one()) {
                    tc::fence_after();
                    tc::mma_tn<KT>(tmem + KT, tmem, sv + b * L::kK, n16, id_o, kt > kk.tile0);
                    tc::commit(bar_o);
                }
                __syncwarp();
            }
            tc::mbar_wait(bar_o, par_o, dead);
            par_o ^= 1;
        }
    } else {
        // ---- softmax
        const uint32_t lane_at = static_cast<uint32_t>(warp * 32) << 16, ts = tmem + lane_at, to = ts + KT;
        const Loader<T, kRows> lq(p.q, p.q_st, p.q_sh, p.dim, head0);
        int par_s = 0, par_o = 0, count = 0;
        bool alive = true;
        for (; more; more = walk.next()) {
            const AttnTile& t = walk.tile;
            const Keys kk = keys_of(t);
            const int rows = kk.rows, row = t.first + tid;
            const bool live = tid < rows;
            int qt = row, qh = 0;  // the row's token in the window, and head
            if (p.pack > 1) qt = row / p.pack, qh = row - qt * p.pack;
            const int64_t token = t.begin + (live ? qt : 0);
            const int head = head0 + (live ? qh : 0);

            float m = -INFINITY, l = 0.0f;  // m: what the weights are taken against
            int2 qp = make_int2(0, 0);
            Range qr{0, 0, 0, 0};
            tc::bar_sync(1, kRows);  // the last tile's staging has been read
            if (kk.tile0 < kk.tile1) {
                if (p.pack == 1)
                    lq.load(sq, kRows, t.begin + t.first, rows, kRows);
                else
                    lq.load_packed(sq, kRows, t.begin, p.q_sh, p.pack, t.first, rows, kRows);
                tc::cp_async_commit();
                if (BIAS) {
                    // rows past the last one take its position: no entry outside the map is looked up
                    qp = bias_pos(p.bias.q_pos, p.bias.axes, t.begin + (t.first + min(tid, rows - 1)) / p.pack);
                    qr = warp_range(qp);
                }
                tc::cp_async_wait<0>();
                tc::fence_async();
                tc::mbar_arrive(bar_q);
            }
            for (int kt = kk.tile0; kt < kk.tile1; ++kt, ++count) {
                const int k0 = kt * KT, n = min(KT, kk.most - k0), n16 = (n + 15) & ~15;
                const KeyPos<KT>* kp = kps + (kBuf == 2 ? count & 1 : 0);
                BiasMode mode = kOne;
                if (BIAS) {
                    alive = tc::mbar_wait(bar_pos(kBuf == 2 ? count & 1 : 0), (count / kBuf) & 1, dead) && alive;
                    mode = bias_mode(p.bias, qr, key_range(kp));
                }
                alive = tc::mbar_wait(bar_s, par_s, dead) && alive;
                par_s ^= 1;
                tc::fence_after();
                // The row's scores, 64 at a time; with more, they are read twice (and, where the bias or the mask
                // changed them, written back between), so that four warps' registers hold them.
                constexpr int kPart = 64, kParts = KT / kPart;
                const bool cut = n != n16 || k0 + n > kk.least;  // some rows see less of the tile
                const int see = live ? (p.causal ? min(qt + kk.shift + 1, t.olen) : t.olen) - k0 : 0;
                float s[kPart];
                float top0 = -INFINITY, top1 = -INFINITY;
#pragma unroll
                for (int h = 0; h < kParts; ++h) {
                    const int h0 = h * kPart;
#pragma unroll
                    for (int c = 0; c < kPart; c += 16)
                        if (h0 + c < n16) tc::tmem_ld16(ts + h0 + c, s + c);
                    tc::wait_ld();
                    if (BIAS) {
#pragma unroll
                        for (int c = 0; c < kPart; c += 16)
                            if (h0 + c < n16)
                                add_bias<KT, 16>(*reinterpret_cast<float(*)[16]>(s + c), c2, p.bias, mode, E + (live ? qh : 0) * entries, kp, h0 + c, qp);
                    }
                    if (cut) {
#pragma unroll
                        for (int c = 0; c < kPart; ++c) s[c] = h0 + c < see ? s[c] : -INFINITY;
                    }
#pragma unroll
                    for (int c = 0; c < kPart; c += 16) {
                        if (h0 + c >= n16) continue;
#pragma unroll
                        for (int i = 0; i < 16; i += 4) {
                            top0 = fmaxf(top0, fmaxf(s[c + i], s[c + i + 1]));
                            top1 = fmaxf(top1, fmaxf(s[c + i + 2], s[c + i + 3]));
                        }
                        if (kParts > 1 && (BIAS || cut)) tc::tmem_st16(ts + h0 + c, s + c);
                    }
                }
                if (kParts > 1 && (BIAS || cut)) tc::wait_st();
                if (BIAS) tc::mbar_arrive(bar_pos_read(kBuf == 2 ? count & 1 : 0));
                // the maximum passes NaN scores by: their weights are NaN whatever m is, and so is the row
                const float top = fmaxf(top0, top1) * (BIAS ? 1.0f : c2);
                const bool rise = top > m + 8.0f || (m == -INFINITY && top > m);
                const float keep = rise ? ex2(m - top) : 1.0f;
                if (rise) m = top;
                if (kt > kk.tile0 && __any_sync(0xffffffffu, rise)) {  // O of the tiles before is there: S came after it
#pragma unroll
                    for (int c = 0; c < DP; c += 16) {
                        if (c >= dim16) continue;
                        float o[16];
                        tc::tmem_ld16(to + c, o);
                        tc::wait_ld();
#pragma unroll
                        for (int i = 0; i < 16; ++i) o[i] *= keep;
                        tc::tmem_st16(to + c, o);
                    }
                }
                // two values an instruction: the scaling and the sum are packed
                const float off = m == -INFINITY ? 0.0f : -m;
                const float2 by = make_float2(BIAS ? 1.0f : c2, BIAS ? 1.0f : c2), off2 = make_float2(off, off);
                float2 sum0 = make_float2(0.0f, 0.0f), sum1 = sum0;
#pragma unroll
                for (int h = 0; h < kParts; ++h) {
                    const int h0 = h * kPart;
                    if (kParts > 1) {
#pragma unroll
                        for (int c = 0; c < kPart; c += 16)
                            if (h0 + c < n16) tc::tmem_ld16(ts + h0 + c, s + c);
                        tc::wait_ld();
                    }
#pragma unroll
                    for (int c = 0; c < kPart; c += 16) {
                        if (h0 + c >= n16) continue;
                        uint32_t w[8];
#pragma unroll
                        for (int i = 0; i < 16; i += 4) {
                            float2 a = make_float2(s[c + i], s[c + i + 1]), b = make_float2(s[c + i + 2], s[c + i + 3]);
                            a = BIAS ? __fadd2_rn(a, off2) : __ffma2_rn(a, by, off2);
                            b = BIAS ? __fadd2_rn(b, off2) : __ffma2_rn(b, by, off2);
                            a.x = ex2(a.x), a.y = ex2(a.y), b.x = ex2(b.x), b.y = ex2(b.y);
                            sum0 = __fadd2_rn(sum0, a);
                            sum1 = __fadd2_rn(sum1, b);
                            w[i / 2] = pack2(a.x, a.y, T{});
                            w[i / 2 + 1] = pack2(b.x, b.y, T{});
                        }
                        tc::tmem_st8(ts + (h0 + c) / 2, w);
                    }
                }
                tc::wait_st();
                tc::fence_before();
                tc::mbar_arrive(bar_p);
                l = l * keep + ((sum0.x + sum0.y) + (sum1.x + sum1.y));
                if (kt + 1 < kk.tile1) par_o ^= 1;  // the warp of the products waits for these
            }
            if (kk.tile0 < kk.tile1) {
                alive = tc::mbar_wait(bar_o, par_o, dead) && alive;
                par_o ^= 1;
                tc::fence_after();
            }
            // O out of tensor memory, staged through the Q panels so that rows are written together
            const float inv = p.splits > 1 ? 1.0f : l == 0.0f ? 0.0f : 1.0f / l;
            const int64_t at = token * p.heads + head;
            const int64_t part = static_cast<int64_t>(blockIdx.z) * p.tq * p.heads + at;
            if (live && p.splits > 1) p.part_ml[2 * part] = m, p.part_ml[2 * part + 1] = l;
            if (live && p.splits == 1 && p.lse != nullptr)
                p.lse[static_cast<int64_t>(head) * p.tq + token] = l == 0.0f ? INFINITY : m + log2f(l);
            bool fine = true;
#pragma unroll
            for (int c = 0; c < DP; c += 16) {
                if (c >= dim16) continue;
                float o[16];
                if (kk.tile0 < kk.tile1) {
                    tc::tmem_ld16(to + c, o);
                    tc::wait_ld();
                } else {
#pragma unroll
                    for (int i = 0; i < 16; ++i) o[i] = 0.0f;
                }
#pragma unroll
                for (int i = 0; i < 16; ++i) fine = fine && (!p.causal || is_finite(o[i]));  // columns past dim are 0
                if (p.splits > 1) {
                    if (live) write_part(p.part_o + part * p.dim, o, c, p.dim);
                } else {
                    stage16<T>(sq, tid, o, c, alive ? inv : __uint_as_float(0x7fffffffu));
                }
            }
            tc::fence_before();  // before the next tile's first P is announced, and so its O is written
            if (p.causal && live && !fine) {
                forward_row<T>(p, token, head, BIAS ? p.bias.k_pos : nullptr, t.obegin, kk.tile0 * KT,
                               min(min(qt + kk.shift + 1, t.olen), kk.tile1 * KT), m == -INFINITY ? 0.0f : m, E + qh * entries, qp, sq,
                               p.splits > 1 ? p.part_o + part * p.dim : nullptr, inv);
            }
            if (p.splits > 1) continue;
            tc::bar_sync(1, kRows);
            store_panel<T, kRows>(sq, p.out, p.heads, p.dim, t.begin, head0, p.pack, t.first, rows);
        }
        if (!alive && tid == 0) count_timeout();
        tc::fence_before();
    }
    __syncthreads();
    if (warp == 0) tc::tmem_free<kCols>(tmem);
}

// ---- tensor maps -------------------------------------------------------------------------
using EncodeTiled = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                                 const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                 CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
EncodeTiled encode_tiled() {
    static const EncodeTiled fn = [] {
        void* f = nullptr;
        cudaDriverEntryPointQueryResult found;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &found) != cudaSuccess ||
            found != cudaDriverEntryPointSuccess)
            return static_cast<EncodeTiled>(nullptr);
        return reinterpret_cast<EncodeTiled>(f);
    }();
    return fn;
}

// A map of [tokens][heads][dim] in boxes of 64 columns and `rows` tokens of one head (columns past dim
// read as 0). False: its strides allow none.
bool tile_map(CUtensorMap* map, int* tokens_y, const void* p, int64_t st, int64_t sh, int dim, int heads, int tokens, int rows, int type) {
    const EncodeTiled encode = encode_tiled();
    if (encode == nullptr || (reinterpret_cast<uintptr_t>(p) & 15) != 0 || st % 8 != 0 || sh % 8 != 0 || st <= 0 || tokens <= 0) return false;
    if (heads == 1 || sh <= 0) {
        if (heads > 1) return false;
        sh = 8 * ((dim + 7) / 8);  // one head: any stride
        if (st % sh != 0) sh = st;
    }
    // the smaller stride first
    *tokens_y = st < sh;
    const int64_t inner = st < sh ? st : sh, outer = st < sh ? sh : st;
    if (outer % inner != 0 || outer * 2 >= (1ll << 40)) return false;
    const cuuint64_t dims[3] = {static_cast<cuuint64_t>(dim), static_cast<cuuint64_t>(*tokens_y ? tokens : heads),
                                static_cast<cuuint64_t>(*tokens_y ? heads : tokens)};
    const cuuint64_t strides[2] = {static_cast<cuuint64_t>(inner * 2), static_cast<cuuint64_t>(outer * 2)};
    const cuuint32_t box[3] = {64, static_cast<cuuint32_t>(*tokens_y ? rows : 1), static_cast<cuuint32_t>(*tokens_y ? 1 : rows)};
    const cuuint32_t one[3] = {1, 1, 1};
    return encode(map, type == kBF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, const_cast<void*>(p), dims,
                  strides, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                  CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <typename T, int KT, int DP, bool BIAS>
cudaError_t fwd_one(const AttnParams& p, cudaStream_t s) {
    const int entries = bias_entries(p.bias);
    const int bytes = 1024 + FwdSmem<KT, DP>::kBytes + 4 * entries * p.pack;
    cudaError_t err = cudaFuncSetAttribute(k_attn_fwd_mma<T, KT, DP, BIAS>, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (err != cudaSuccess) return err;
    TileMaps maps;
    maps.use = p.dim % 8 == 0 &&
               tile_map(&maps.k, &maps.k_tokens_y, p.k, p.k_st, p.k_sh, p.dim, p.kv_heads, p.tk, KT, kIsBf16<T> ? kBF16 : kF16) &&
               tile_map(&maps.v, &maps.v_tokens_y, p.v, p.v_st, p.v_sh, p.dim, p.kv_heads, p.tk, KT, kIsBf16<T> ? kBF16 : kF16);
    // Blocks stay for several tiles of one head; four rounds of them even out tiles of unequal
    // length, one where each has to expand a bias first.
    const int groups = p.heads / p.pack, resident = 148 * (KT == 64 ? 3 : 2) * (BIAS ? 1 : 4);
    const int slots = attn_slots(static_cast<int64_t>(p.tq) * p.pack, p.windows, kRows);
    const int per_head = (resident + groups * p.splits - 1) / (groups * p.splits);
    k_attn_fwd_mma<T, KT, DP, BIAS><<<dim3(slots < per_head ? slots : per_head, groups, p.splits), kRows + 32, bytes, s>>>(p, maps);
    return cudaGetLastError();
}
template <typename T>
cudaError_t fwd_type(const AttnParams& p, cudaStream_t s) {
    if (p.bias.table != nullptr) return p.dim <= 64 ? fwd_one<T, 64, 64, true>(p, s) : fwd_one<T, 128, 128, true>(p, s);
    return p.dim <= 64 ? fwd_one<T, 64, 64, false>(p, s) : fwd_one<T, 128, 128, false>(p, s);
}

}  // namespace

cudaError_t launch_attn_forward_mma(const AttnParams& p, int type, cudaStream_t s) {
    return type == kBF16 ? fwd_type<__nv_bfloat16>(p, s) : fwd_type<__half>(p, s);
}

cudaError_t attn_timeouts(unsigned int* count) {
    return cudaMemcpyFromSymbol(count, g_timeouts, sizeof(unsigned int));
}

}  // namespace oss
