// Window attention of 16-bit types on the tensor cores (tcgen05): forward.
//
// A block of 128 threads holds 128 query rows (thread = row = tensor-memory lane) and walks its
// window's keys KT at a time:
//   S = Q K^T into tensor memory (both operands from shared memory)
//   each thread reads its row of S, keeps the running maximum and sum in registers, and writes
//   the weights back over S as 16-bit values
//   O += P V, P from tensor memory
// K of the next tile is fetched while the softmax runs, V while S is computed, so that one buffer
// of each is enough; two to four blocks share an SM and fill each other's waits. Tiles end at
// the window's last key rounded up to 16, whatever KT is: N of S and K of P V are set by it.
// The running maximum that the weights are taken against moves only when a row exceeds it by
// 2^8: O has to be scaled in tensor memory then, which after the first tiles hardly happens.
// With head dims up to 64 the exponentials (16 a clock and SM) bound long windows: 64-key tiles
// leave room for four blocks (128 of 512 tensor-memory columns each). With 128 the products do,
// and 128-key tiles feed them from shared memory at the full rate.
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
    static constexpr int kQ = kRows * DP * 2, kK = KT * DP * 2;
    static constexpr int kBytes = kQ + 2 * kK + static_cast<int>(sizeof(KeyPos<KT>)) + 64 + 4 * static_cast<int>(sizeof(Range));
};

template <typename T, int KT, int DP, bool BIAS>
__global__ void __launch_bounds__(kRows, KT == 64 ? 4 : 2) k_attn_fwd_mma(const __grid_constant__ AttnParams p) {
    using L = FwdSmem<KT, DP>;
    constexpr int kCols = KT + DP;  // 128 or 256: S (P over it), then O
    constexpr int kBf16 = std::is_same<T, __nv_bfloat16>::value ? 1 : 0;
    extern __shared__ __align__(16) unsigned char smem_raw[];
    unsigned char* base = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    const uint32_t sq = tc::smem_addr(base), sk = sq + L::kQ, sv = sk + L::kK;
    KeyPos<KT>* kp = reinterpret_cast<KeyPos<KT>*>(base + L::kQ + 2 * L::kK);
    Range* qrange = reinterpret_cast<Range*>(kp + 1);
    uint64_t* bars = reinterpret_cast<uint64_t*>(qrange + 4);
    uint32_t* slot_tmem = reinterpret_cast<uint32_t*>(bars + 2);
    float* E = reinterpret_cast<float*>(bars + 8);
    const uint32_t bar_s = tc::smem_addr(bars), bar_o = bar_s + 8;

    const int tid = threadIdx.x, warp = tid >> 5;
    const int head0 = blockIdx.y * p.pack, kvh = head0 / (p.heads / p.kv_heads);
    const int entries = BIAS ? bias_entries(p.bias) : 0, dim16 = (p.dim + 15) & ~15;
    const Loader<T, kRows> lq(p.q, p.q_st, p.q_sh, p.dim, head0), lk(p.k, p.k_st, p.k_sh, p.dim, kvh),
        lv(p.v, p.v_st, p.v_sh, p.dim, kvh);
    const float c2 = p.scale * kLog2e;

    const int slots = attn_slots(static_cast<int64_t>(p.tq) * p.pack, p.windows, kRows);
    const int chunk = (slots + gridDim.x - 1) / gridDim.x;
    // causal windows: the last tiles see the most keys and go first
    const int slot0 = (p.causal ? gridDim.x - 1 - blockIdx.x : blockIdx.x) * chunk;
    AttnWalk walk;
    bool more = walk.start(p.q_off, p.tq, p.k_off, p.tk, p.windows, p.pack, kRows, slot0, min(slots, slot0 + chunk), p.tiny_max);
    if (!more) return;

    if (tid == 0) {
        tc::mbar_init(bar_s, 1);
        tc::mbar_init(bar_o, 1);
        tc::mbar_init_fence();
    }
    if (warp == 0) tc::tmem_alloc<kCols>(tc::smem_addr(slot_tmem));
    if constexpr (BIAS)
        for (int e = tid; e < entries * p.pack; e += kRows) E[e] = bias_entry(p.bias, p.heads, head0 + e / entries, e % entries);
    tc::fence_before();
    __syncthreads();
    tc::fence_after();
    const uint32_t tmem = *slot_tmem, lane_at = static_cast<uint32_t>(warp * 32) << 16;
    const uint32_t ts = tmem + lane_at, to = ts + KT;
    const uint32_t id_o = tc::idesc(kBf16, dim16, false, true);
    int par_s = 0, par_o = 0;  // parities of the next wait
    bool alive = true;

    for (; more; more = walk.next()) {
        const AttnTile& t = walk.tile;
        const int rows = min(kRows, t.len * p.pack - t.first);
        const int row = t.first + tid;
        const bool live = tid < rows;
        int qt = row, qh = 0;  // the row's token in the window, and head
        if (p.pack > 1) qt = row / p.pack, qh = row - qt * p.pack;
        const int shift = t.olen - t.len;
        int most = t.olen, least = t.olen;  // keys that the last row sees, and the first
        if (p.causal) {
            most = min(max((p.pack > 1 ? (t.first + rows - 1) / p.pack : t.first + rows - 1) + shift + 1, 0), t.olen);
            least = min(max((p.pack > 1 ? t.first / p.pack : t.first) + shift + 1, 0), t.olen);
        }
        int tile0 = 0, tile1 = (most + KT - 1) / KT;
        if (p.splits > 1) {
            const int per = (tile1 + p.splits - 1) / p.splits;
            tile0 = min(static_cast<int>(blockIdx.z) * per, tile1);
            tile1 = min(tile0 + per, tile1);
        }
        const int64_t token = t.begin + (live ? qt : 0);
        const int head = head0 + (live ? qh : 0);

        float m = -INFINITY, l = 0.0f;  // m: what the weights are taken against
        int2 qp = make_int2(0, 0);
        __syncthreads();  // the last tile's staging has been read
        if (tile0 < tile1) {
            const int k0 = tile0 * KT, n = min(KT, most - k0), n16 = (n + 15) & ~15;
            if (p.pack == 1)
                lq.load(sq, kRows, t.begin + t.first, rows, kRows);
            else
                lq.load_packed(sq, kRows, t.begin, p.q_sh, p.pack, t.first, rows, kRows);
            lk.load(sk, KT, t.obegin + k0, n, n16);
            tc::cp_async_commit();
            lv.load(sv, KT, t.obegin + k0, n, n16);
            tc::cp_async_commit();
            if (BIAS) {
                load_key_pos<KT>(kp, p.bias, t.obegin + k0, n);
                // rows past the last one take its position: no entry outside the map is looked up
                qp = bias_pos(p.bias.q_pos, p.bias.axes, t.begin + (t.first + min(tid, rows - 1)) / p.pack);
                const Range r = warp_range(qp);
                if ((tid & 31) == 0) qrange[warp] = r;
            }
        }
        for (int kt = tile0; kt < tile1; ++kt) {
            const int k0 = kt * KT, n = min(KT, most - k0), n16 = (n + 15) & ~15;
            if (kt == tile0)
                tc::cp_async_wait<1>();
            else
                tc::cp_async_wait<0>();
            tc::fence_async();
            tc::fence_before();
            __syncthreads();
            if (kt > tile0) {  // O of the tile before: P and V are free
                alive = tc::mbar_wait(bar_o, par_o) && alive;
                par_o ^= 1;
            }
            if (tid == 0) {
                tc::fence_after();
                tc::mma_nt<DP, kRows, KT>(tmem, sq, sk, dim16, tc::idesc(kBf16, n16, false, false));
                tc::commit(bar_s);
            }
            if (kt > tile0) {
                lv.load(sv, KT, t.obegin + k0, n, n16);
                tc::cp_async_commit();
            }
            BiasMode mode = kOne;
            if (BIAS) mode = bias_mode(p.bias, join(join(qrange[0], qrange[1]), join(qrange[2], qrange[3])), key_range(kp));
            alive = tc::mbar_wait(bar_s, par_s) && alive;
            par_s ^= 1;
            tc::fence_after();
            // the row's scores
            float s[KT];
#pragma unroll
            for (int c = 0; c < KT; c += 16)
                if (c < n16) tc::tmem_ld16(ts + c, s + c);
            if (kt + 1 < tile1) {
                const int n2 = min(KT, most - k0 - KT);
                lk.load(sk, KT, t.obegin + k0 + KT, n2, (n2 + 15) & ~15);
            }
            tc::cp_async_commit();  // a group for each tile, an empty one after the last
            tc::wait_ld();
            if (BIAS) {
#pragma unroll
                for (int c = 0; c < KT; c += 16)
                    if (c < n16) add_bias<KT, 16>(*reinterpret_cast<float(*)[16]>(s + c), c2, p.bias, mode, E + (live ? qh : 0) * entries, kp, c, qp);
            }
            if (n != n16 || k0 + n > least) {  // some rows see less of the tile
                const int see = live ? (p.causal ? min(qt + shift + 1, t.olen) : t.olen) - k0 : 0;
#pragma unroll
                for (int c = 0; c < KT; ++c) s[c] = c < see ? s[c] : -INFINITY;
            }
            float top = -INFINITY;
#pragma unroll
            for (int c = 0; c < KT; c += 16) {
                if (c >= n16) continue;
#pragma unroll
                for (int i = 0; i < 16; i += 2) top = fmaxf(top, fmaxf(s[c + i], s[c + i + 1]));
            }
            // the maximum passes NaN scores by: their weights are NaN whatever m is, and so is the row
            if (!BIAS) top *= c2;
            const bool rise = top > m + 8.0f || (m == -INFINITY && top > m);
            const float keep = rise ? ex2(m - top) : 1.0f;
            if (rise) m = top;
            if (kt > tile0 && __any_sync(0xffffffffu, rise)) {
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
                tc::tmem_st8(ts + c / 2, w);
            }
            l = l * keep + ((sum0.x + sum0.y) + (sum1.x + sum1.y));
            tc::wait_st();
            tc::cp_async_wait<1>();  // V of this tile
            tc::fence_async();
            tc::fence_before();
            __syncthreads();
            if (tid == 0) {
                tc::fence_after();
                tc::mma_tn<KT>(tmem + KT, tmem, sv, n16, id_o, kt > tile0);
                tc::commit(bar_o);
            }
            if (BIAS && kt + 1 < tile1) load_key_pos<KT>(kp, p.bias, t.obegin + k0 + KT, min(KT, most - k0 - KT));
        }
        if (tile0 < tile1) {
            alive = tc::mbar_wait(bar_o, par_o) && alive;
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
            if (tile0 < tile1) {
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
        if (p.causal && live && !fine) {
            forward_row<T>(p, token, head, BIAS ? p.bias.k_pos : nullptr, t.obegin, tile0 * KT,
                           min(min(qt + shift + 1, t.olen), tile1 * KT), m == -INFINITY ? 0.0f : m, E + qh * entries, qp, sq,
                           p.splits > 1 ? p.part_o + part * p.dim : nullptr, inv);
        }
        if (p.splits > 1) continue;
        __syncthreads();
        store_panel<T, kRows>(sq, p.out, p.heads, p.dim, t.begin, head0, p.pack, t.first, rows);
    }
    if (!alive && tid == 0) count_timeout();
    tc::fence_before();
    __syncthreads();
    if (warp == 0) tc::tmem_free<kCols>(tmem);
}

template <typename T, int KT, int DP, bool BIAS>
cudaError_t fwd_one(const AttnParams& p, cudaStream_t s) {
    const int entries = bias_entries(p.bias);
    const int bytes = 1024 + FwdSmem<KT, DP>::kBytes + 4 * entries * p.pack;
    cudaError_t err = cudaFuncSetAttribute(k_attn_fwd_mma<T, KT, DP, BIAS>, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (err != cudaSuccess) return err;
    // Blocks stay for several tiles of one head; four rounds of them even out tiles of unequal
    // length, one where each has to expand a bias first.
    const int groups = p.heads / p.pack, resident = 148 * (KT == 64 ? 4 : 2) * (BIAS ? 1 : 4);
    const int slots = attn_slots(static_cast<int64_t>(p.tq) * p.pack, p.windows, kRows);
    const int per_head = (resident + groups * p.splits - 1) / (groups * p.splits);
    k_attn_fwd_mma<T, KT, DP, BIAS><<<dim3(slots < per_head ? slots : per_head, groups, p.splits), kRows, bytes, s>>>(p);
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
