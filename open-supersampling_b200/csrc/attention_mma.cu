// Window attention of 16-bit types on the tensor cores (tcgen05): forward.
//
// A block holds 128 query rows and walks its window's keys 64 at a time. Four warps do the softmax
// (thread = row = tensor-memory lane), one issues the products, one moves keys and values:
//   S = Q K^T into tensor memory (both operands from shared memory)
//   each thread reads its row of S, keeps the running maximum and sum in registers, and writes
//   the weights back over S as 16-bit values
//   O += P V, P from tensor memory
// S of the next tile is computed into a second buffer while the softmax runs, and two blocks share an
// SM, so that the exponentials (16 a clock and SM) hardly pause. Keys and values arrive by tensor
// copies, two tiles ahead; 16- or 4-byte copies or plain loads where strides or alignment allow none.
// One causal window of 16320, 8 heads over 2 of 128: 686 us, 796 TFLOP/s of the formula's products (a single buffer
// of S and keys loaded by the softmax warps took 975 us). Products and softmax wait for one another: S of a tile for
// P V of two tiles before, the softmax for O of the one before; the tensor pipe, the exponentials and the issue
// slots are each less than half taken. 68 single tokens over 8160 keys, split: 94 us, 3.4 TB/s of keys and values.
// Tiles end at the window's last key rounded up to 16: N of S and K of P V are set by it.
// The running maximum that the weights are taken against moves only when a row exceeds it by
// 2^8: O has to be scaled in tensor memory then, which after the first tiles hardly happens.
#include <cuda.h>

#include "attention_mma.cuh"
#include "internal.h"

namespace oss {
namespace {

// ---- a row again, where a product met what its mask hides --------------------------------
// Sums a row over the keys that it sees, in the order of its tiles.
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
template <int DP>
struct FwdSmem {
    static constexpr int KT = 64;
    static constexpr int kQ = kRows * DP * 2, kK = KT * DP * 2;
    static constexpr int kTiles = kQ + 4 * kK;  // two of keys, two of values
    static constexpr int kBytes = kTiles + 2 * static_cast<int>(sizeof(KeyPos<KT>)) + 192;
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

// REST, for training: what rounding takes from the weights follows them as 16-bit values in the other half of
// their buffer, O takes both, and what rounding takes from out is written too. dout . out of the backward is
// then right to fp32: with rounded weights the table's gradient of packed causal histories was off by up to
// 1.7 times what its own rounding makes it. 7 windows of up to 4095 tokens, forward and backward: 10% of the time.
template <typename T, int DP, bool BIAS, bool REST>
__global__ void __launch_bounds__(kRows + 64, 2) k_attn_fwd_mma(const __grid_constant__ AttnParams p, const __grid_constant__ TileMaps maps) {
    using L = FwdSmem<DP>;
    constexpr int KT = L::KT, kCols = 256, kS = 64, kO = 128;  // columns: S (P over it) twice, then O
    constexpr int kThreads = kRows + 64;
    constexpr int kBf16 = std::is_same<T, __nv_bfloat16>::value ? 1 : 0;
    extern __shared__ __align__(16) unsigned char smem_raw[];
    unsigned char* base = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    const uint32_t sq = tc::smem_addr(base), sk = sq + L::kQ, sv = sk + 2 * L::kK;
    KeyPos<KT>* kps = reinterpret_cast<KeyPos<KT>*>(base + L::kTiles);
    uint64_t* bars = reinterpret_cast<uint64_t*>(kps + 2);
    uint32_t* slot_tmem = reinterpret_cast<uint32_t*>(bars + 20);
    volatile int* dead = reinterpret_cast<volatile int*>(bars + 21);
    float* E = reinterpret_cast<float*>(bars + 24);
    // Barriers. One each: Q there, O done. For each buffer: P there (a softmax warp may be a tile ahead of
    // another), S done, keys there and read, values there and read, key positions there and read. The last one is
    // for products in flight after a wait that ran out.
    const uint32_t bar0 = tc::smem_addr(bars), bar_q = bar0, bar_o = bar0 + 8, bar_p = bar0 + 16, bar_s = bar0 + 32, bar_k = bar0 + 48,
                   bar_k_read = bar0 + 64, bar_v = bar0 + 80, bar_v_read = bar0 + 96, bar_pos = bar0 + 112, bar_pos_read = bar0 + 128, bar_end = bar0 + 144;

    const int tid = threadIdx.x, warp = tid >> 5;
    const int head0 = blockIdx.y * p.pack, kvh = head0 / (p.heads / p.kv_heads);
    const int entries = BIAS ? bias_entries(p.bias) : 0, dim16 = (p.dim + 15) & ~15;
    const float c2 = p.scale * kLog2e;

    const int slots = attn_slots(static_cast<int64_t>(p.tq) * p.pack, p.windows, kRows);
    const int chunk = (slots + gridDim.x - 1) / gridDim.x;
    // causal windows: the last tiles see the most keys and go first
    const int slot0 = (p.causal ? gridDim.x - 1 - blockIdx.x : blockIdx.x) * chunk;
    AttnWalk<kRows> walk;
    bool more = walk.start(p.q_off, p.tq, p.k_off, p.tk, p.windows, p.pack, slot0, min(slots, slot0 + chunk), p.tiny_max);
    if (!more) return;

    if (tid == 0) {
        for (int b = 0; b < 19; ++b) tc::mbar_init(bar0 + 8 * b, b == 0 || b == 2 || b == 3 || b == 16 || b == 17 ? kRows : 1);
        tc::mbar_init_fence();
        *dead = 0;
    }
    if (warp == 0) tc::tmem_alloc<kCols>(tc::smem_addr(slot_tmem));
    if constexpr (BIAS)
        for (int e = tid; e < entries * p.pack; e += kThreads) E[e] = bias_entry(p.bias, p.heads, head0 + e / entries, e % entries);
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

    // Every role counts the tiles of keys that it has passed: tile number u is in buffer u & 1, its barriers in
    // their phase u >> 1.
    int u = 0;
    if (warp == 5) {
        // ---- keys and values
        const int lane = tid & 31, panels = dim16 > 64 ? 2 : 1;
        bool ok = true;
        int k_sent = 0, v_sent = 0;  // tiles whose copies have been issued
        for (; ok && more; more = walk.next()) {
            const AttnTile& t = walk.tile;
            const Keys kk = keys_of(t);
            for (int kt = kk.tile0; kt < kk.tile1; ++kt, ++u) {
                const int b = u & 1, parity = (u >> 1) & 1, n = min(KT, kk.most - kt * KT), token = t.obegin + kt * KT;
                // of two tiles before: passes at once at first
                if (!(ok = __all_sync(0xffffffffu, tc::mbar_wait(bar_k_read + 8 * b, parity ^ 1, dead)))) break;
                if (maps.use) {
                    if (tc::elect_one()) {
                        tc::mbar_expect(bar_k + 8 * b, panels * KT * 128);
                        for (int h = 0; h < panels; ++h)
                            tc::tma_load(sk + b * L::kK + h * KT * 128, &maps.k, bar_k + 8 * b, 64 * h, maps.k_tokens_y ? token : kvh,
                                         maps.k_tokens_y ? kvh : token);
                    }
                    ++k_sent;
                } else {
                    warp_load<T>(sk + b * L::kK, KT, p.k, p.k_st, p.k_sh, p.dim, kvh, token, n, (n + 15) & ~15);
                }
                if (!(ok = __all_sync(0xffffffffu, tc::mbar_wait(bar_v_read + 8 * b, parity ^ 1, dead)))) break;
                if (maps.use) {
                    if (tc::elect_one()) {
                        tc::mbar_expect(bar_v + 8 * b, panels * KT * 128);
                        for (int h = 0; h < panels; ++h)
                            tc::tma_load(sv + b * L::kK + h * KT * 128, &maps.v, bar_v + 8 * b, 64 * h, maps.v_tokens_y ? token : kvh,
                                         maps.v_tokens_y ? kvh : token);
                    }
                    ++v_sent;
                } else {
                    warp_load<T>(sv + b * L::kK, KT, p.v, p.v_st, p.v_sh, p.dim, kvh, token, n, (n + 15) & ~15);
                    tc::cp_async_commit();
                    tc::cp_async_wait<0>();
                    tc::fence_async();
                    __syncwarp();
                    if (lane == 0) {
                        tc::mbar_arrive(bar_k + 8 * b);
                        tc::mbar_arrive(bar_v + 8 * b);
                    }
                }
                if (BIAS) {
                    if (!(ok = __all_sync(0xffffffffu, tc::mbar_wait(bar_pos_read + 8 * b, parity ^ 1, dead)))) break;
                    load_key_pos_warp<KT>(kps + b, p.bias, token, n);
                    __syncwarp();
                    if (lane == 0) tc::mbar_arrive(bar_pos + 8 * b);
                }
            }
            if (!ok) break;
        }
        if (!ok) {  // the copies in flight, before the block may end
            tc::cp_async_commit();
            tc::cp_async_wait<0>();
            for (int i = max(k_sent - 2, 0); i < k_sent; ++i) tc::mbar_settle(bar_k + 8 * (i & 1), (i >> 1) & 1);
            for (int i = max(v_sent - 2, 0); i < v_sent; ++i) tc::mbar_settle(bar_v + 8 * (i & 1), (i >> 1) & 1);
        }
    } else if (warp == 4) {
        // ---- products
        const int lane = tid & 31;
        const uint32_t id_o = tc::idesc(kBf16, dim16, false, true);
        int par_q = 0, par_o = 0;
        bool ok = true;  // no wait has run out: whatever is issued has its operands
        auto wait = [&](uint32_t bar, int parity) { return ok = ok && __all_sync(0xffffffffu, tc::mbar_wait(bar, parity, dead)); };
        for (; ok && more; more = walk.next()) {
            const Keys kk = keys_of(walk.tile);
            if (kk.tile0 >= kk.tile1) continue;
            // S of tile kt, number v
            auto scores = [&](int kt, int v) {
                const int b = v & 1, n16 = (min(KT, kk.most - kt * KT) + 15) & ~15;
                if (!wait(bar_k + 8 * b, (v >> 1) & 1)) return;
                if (tc::elect_one()) {
                    tc::fence_after();
                    tc::mma_nt<DP, kRows, KT>(tmem + b * kS, sq, sk + b * L::kK, dim16, tc::idesc(kBf16, n16, false, false));
                    tc::commit(bar_s + 8 * b);
                    tc::commit(bar_k_read + 8 * b);
                }
                __syncwarp();
            };
            if (!wait(bar_q, par_q)) break;
            par_q ^= 1;
            scores(kk.tile0, u);
            for (int kt = kk.tile0; ok && kt < kk.tile1; ++kt, ++u) {
                const int b = u & 1, n = min(KT, kk.most - kt * KT), n16 = (n + 15) & ~15;
                if (kt > kk.tile0) {  // P of the tile before has been read: its buffer takes the next S
                    if (!wait(bar_o, par_o)) break;
                    par_o ^= 1;
                }
                if (kt + 1 < kk.tile1) scores(kt + 1, u + 1);
                if (!wait(bar_v + 8 * b, (u >> 1) & 1)) break;
                if (maps.use && n < n16) {  // what follows the window's last value meets weights of 0: it must not be NaN
                    const int chunks = dim16 / 8;
                    for (int i = lane; i < (n16 - n) * chunks; i += 32) {
                        const int r = n + i / chunks, c = i % chunks;
                        Loader<T, 32>::store_zero(sv + b * L::kK + (c >> 3) * KT * 128 + r * 128 + (((c & 7) ^ (r & 7)) << 4));
                    }
                    tc::fence_async();
                    __syncwarp();
                }
                if (!wait(bar_p + 8 * b, (u >> 1) & 1)) break;
                if (tc::elect_one()) {
                    tc::fence_after();
                    tc::mma_tn<KT>(tmem + kO, tmem + b * kS, sv + b * L::kK, n16, id_o, kt > kk.tile0);
                    if (REST) tc::mma_tn<KT>(tmem + kO, tmem + b * kS + KT / 2, sv + b * L::kK, n16, id_o, true);
                    tc::commit(bar_o);
                    tc::commit(bar_v_read + 8 * b);
                }
                __syncwarp();
            }
            if (!wait(bar_o, par_o)) break;
            par_o ^= 1;
        }
        if (!ok) {  // the products in flight, before their tensor memory is freed
            if (tc::elect_one()) tc::commit(bar_end);
            __syncwarp();
            tc::mbar_settle(bar_end, 0);
        }
    } else {
        // ---- softmax
        const uint32_t lane_at = static_cast<uint32_t>(warp * 32) << 16, to = tmem + lane_at + kO;
        const Loader<T, kRows> lq(p.q, p.q_st, p.q_sh, p.dim, head0);
        int par_o = 0;  // phase of O of the tile before
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
            for (int kt = kk.tile0; kt < kk.tile1; ++kt, ++u) {
                const int b = u & 1, k0 = kt * KT, n = min(KT, kk.most - k0), n16 = (n + 15) & ~15;
                const uint32_t ts = tmem + lane_at + b * kS;
                const KeyPos<KT>* kp = kps + b;
                BiasMode mode = kOne;
                if (BIAS) {
                    alive = tc::mbar_wait(bar_pos + 8 * b, (u >> 1) & 1, dead) && alive;
                    mode = bias_mode(p.bias, qr, key_range(kp));
                }
                alive = tc::mbar_wait(bar_s + 8 * b, (u >> 1) & 1, dead) && alive;
                tc::fence_after();
                float s[KT];
#pragma unroll
                for (int c = 0; c < KT; c += 16)
                    if (c < n16) tc::tmem_ld16(ts + c, s + c);
                tc::wait_ld();
                if (BIAS) {
                    add_bias<KT>(s, c2, p.bias, mode, E + (live ? qh : 0) * entries, kp, 0, n16, qp);
                    tc::mbar_arrive(bar_pos_read + 8 * b);
                }
                if (n != KT || k0 + n > kk.least) {  // some rows see less of the tile
                    const int see = live ? (p.causal ? min(qt + kk.shift + 1, t.olen) : t.olen) - k0 : 0;
#pragma unroll
                    for (int c = 0; c < KT; ++c) s[c] = c < see ? s[c] : -INFINITY;
                }
                float top0 = -INFINITY, top1 = -INFINITY;
#pragma unroll
                for (int c = 0; c < KT; c += 4) {
                    top0 = fmaxf(top0, fmaxf(s[c], s[c + 1]));
                    top1 = fmaxf(top1, fmaxf(s[c + 2], s[c + 3]));
                }
                // the maximum passes NaN scores by: their weights are NaN whatever m is, and so is the row
                const float top = fmaxf(top0, top1) * (BIAS ? 1.0f : c2);
                const bool rise = top > m + 8.0f || (m == -INFINITY && top > m);
                const float keep = rise ? ex2(m - top) : 1.0f;
                if (rise) m = top;
                const bool scaled = kt > kk.tile0 && __any_sync(0xffffffffu, rise);
                if (scaled) {
                    alive = tc::mbar_wait(bar_o, par_o, dead) && alive;
                    tc::fence_after();
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
                for (int c = 0; c < KT; c += 16) {
                    if (c >= n16) continue;
                    uint32_t w[8];
                    float rest[16];
#pragma unroll
                    for (int i = 0; i < 16; i += 4) {
                        float2 x = make_float2(s[c + i], s[c + i + 1]), y = make_float2(s[c + i + 2], s[c + i + 3]);
                        x = BIAS ? __fadd2_rn(x, off2) : __ffma2_rn(x, by, off2);
                        y = BIAS ? __fadd2_rn(y, off2) : __ffma2_rn(y, by, off2);
                        x.x = ex2(x.x), x.y = ex2(x.y), y.x = ex2(y.x), y.y = ex2(y.y);
                        sum0 = __fadd2_rn(sum0, x);
                        sum1 = __fadd2_rn(sum1, y);
                        w[i / 2] = pack2(x.x, x.y, T{});
                        w[i / 2 + 1] = pack2(y.x, y.y, T{});
                        if (REST) {
                            rest[i] = lost_by<T>(x.x), rest[i + 1] = lost_by<T>(x.y);
                            rest[i + 2] = lost_by<T>(y.x), rest[i + 3] = lost_by<T>(y.y);
                        }
                    }
                    tc::tmem_st8(ts + c / 2, w);
                    if (REST) {
#pragma unroll
                        for (int i = 0; i < 8; ++i) w[i] = pack2(rest[2 * i], rest[2 * i + 1], T{});
                        tc::tmem_st8(ts + KT / 2 + c / 2, w);
                    }
                }
                tc::wait_st();
                if (kt > kk.tile0) {
                    // O of the tile before. S runs ahead of O: seen only after this tile's weights are announced, its
                    // phase could be told neither from the one before nor from the next.
                    if (!scaled) alive = tc::mbar_wait(bar_o, par_o, dead) && alive;
                    par_o ^= 1;
                }
                tc::fence_before();
                tc::mbar_arrive(bar_p + 8 * b);
                l = l * keep + ((sum0.x + sum0.y) + (sum1.x + sum1.y));
            }
            if (kk.tile0 < kk.tile1) {
                alive = tc::mbar_wait(bar_o, par_o, dead) && alive;
                par_o ^= 1;
                tc::fence_after();
            }
            // A wait of the block has run out: its rows become NaN. (The warps that load and issue stop at theirs,
            // and every wait for them then runs out here too.)
            alive = alive && *dead == 0;
            if (!alive) l = __uint_as_float(0x7fffffffu);
            // O out of tensor memory, staged through the Q panels so that rows are written together
            const float inv = p.splits > 1 ? (alive ? 1.0f : l) : l == 0.0f ? 0.0f : 1.0f / l;
            const int64_t at = token * p.heads + head;
            const int64_t part = static_cast<int64_t>(blockIdx.z) * p.tq * p.heads + at;
            if (live && p.splits > 1) p.part_ml[2 * part] = m, p.part_ml[2 * part + 1] = l;
            if (live && p.splits == 1 && p.lse != nullptr)
                store_lse(p, static_cast<int64_t>(head) * p.tq + token, m, l);
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
                    if (!alive)
#pragma unroll
                        for (int i = 0; i < 16; ++i) o[i] = l;
                    if (live) write_part(p.part_o + part * p.dim, o, c, p.dim);
                } else {
                    stage16<T>(sq, tid, o, c, inv);
                }
            }
            tc::fence_before();  // before the next tile's first P is announced, and so its O is written
            // Where l is finite, so is every weight: the values are at fault.
            bool again = p.causal && live && alive && !fine && is_finite(l);
            if (__any_sync(0xffffffffu, again)) {
                const int lo = kk.tile0 * KT, hi = min(kk.most, kk.tile1 * KT), see = min(max(qt + kk.shift + 1, lo), hi);
                const T* vb = static_cast<const T*>(p.v) + t.obegin * p.v_st + kvh * p.v_sh;
                const int last = last_not_finite<T>(vb, p.v_st, __reduce_min_sync(0xffffffffu, again ? see : hi), hi, p.dim);
                again = again && last >= see && hidden_spoils<T>(vb, p.v_st, see, last + 1, lo, see, p.dim);
                if (again)
                    forward_row<T>(p, token, head, BIAS ? p.bias.k_pos : nullptr, t.obegin, lo, see, m == -INFINITY ? 0.0f : m, E + qh * entries,
                                   qp, sq, p.splits > 1 ? p.part_o + part * p.dim : nullptr, inv);
            }
            if (p.splits > 1) continue;
            tc::bar_sync(1, kRows);
            store_panel<T, kRows>(sq, p.out, p.heads, p.dim, t.begin, head0, p.pack, t.first, rows);
            if (!REST) continue;
            tc::bar_sync(1, kRows);  // the staging has been read
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
                for (int i = 0; i < 16; ++i) o[i] = fine ? lost_by<T>(o[i] * inv) : 0.0f;
                stage16<T>(sq, tid, o, c, 1.0f);
            }
            tc::fence_before();
            tc::bar_sync(1, kRows);
            store_panel<T, kRows>(sq, p.out_lo, p.heads, p.dim, t.begin, head0, p.pack, t.first, rows);
        }
        tc::fence_before();
    }
    __syncthreads();
    if (tid == 0 && *dead != 0) count_timeout();
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

template <typename T, int DP, bool BIAS, bool REST>
cudaError_t fwd_one(const AttnParams& p, cudaStream_t s) {
    const int entries = bias_entries(p.bias);
    const int bytes = 1024 + FwdSmem<DP>::kBytes + 4 * entries * p.pack;
    cudaError_t err = allow_smem(k_attn_fwd_mma<T, DP, BIAS, REST>);
    if (err != cudaSuccess) return err;
    const int type = kIsBf16<T> ? kBF16 : kF16;
    TileMaps maps;
    maps.use = p.dim % 8 == 0 && tile_map(&maps.k, &maps.k_tokens_y, p.k, p.k_st, p.k_sh, p.dim, p.kv_heads, p.tk, 64, type) &&
               tile_map(&maps.v, &maps.v_tokens_y, p.v, p.v_st, p.v_sh, p.dim, p.kv_heads, p.tk, 64, type);
    // Blocks stay for several tiles of one head; four rounds of them even out tiles of unequal
    // length, one where each has to expand a bias first.
    const int groups = p.heads / p.pack, resident = 148 * 2 * (BIAS ? 1 : 4);
    const int slots = attn_slots(static_cast<int64_t>(p.tq) * p.pack, p.windows, kRows);
    const int per_head = (resident + groups * p.splits - 1) / (groups * p.splits);
    k_attn_fwd_mma<T, DP, BIAS, REST><<<dim3(slots < per_head ? slots : per_head, groups, p.splits), kRows + 64, bytes, s>>>(p, maps);
    return cudaGetLastError();
}
template <typename T, bool REST>
cudaError_t fwd_rest(const AttnParams& p, cudaStream_t s) {
    if (p.bias.table != nullptr) return p.dim <= 64 ? fwd_one<T, 64, true, REST>(p, s) : fwd_one<T, 128, true, REST>(p, s);
    return p.dim <= 64 ? fwd_one<T, 64, false, REST>(p, s) : fwd_one<T, 128, false, REST>(p, s);
}
template <typename T>
cudaError_t fwd_type(const AttnParams& p, cudaStream_t s) {
    return p.out_lo != nullptr ? fwd_rest<T, true>(p, s) : fwd_rest<T, false>(p, s);
}

}  // namespace

cudaError_t launch_attn_forward_mma(const AttnParams& p, int type, cudaStream_t s) {
    return type == kBF16 ? fwd_type<__nv_bfloat16>(p, s) : fwd_type<__half>(p, s);
}

cudaError_t attn_timeouts(unsigned int* count) {
    return cudaMemcpyFromSymbol(count, g_timeouts, sizeof(unsigned int));
}

}  // namespace oss
