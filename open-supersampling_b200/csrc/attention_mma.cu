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

template <typename T, int KT, int DP>
__global__ void __launch_bounds__(kRows, KT == 64 ? 4 : 2) k_attn_fwd_mma(const __grid_constant__ AttnParams p) {
    using L = FwdSmem<KT, DP>;
    constexpr int kCols = KT + DP;  // 128 or 256: S (P over it), then O
    constexpr int kBf16 = sizeof(T) == 2 && std::is_same<T, __nv_bfloat16>::value ? 1 : 0;
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
    const int entries = bias_entries(p.bias), dim16 = (p.dim + 15) & ~15;
    const int slots = attn_slots(static_cast<int64_t>(p.tq) * p.pack, p.windows, kRows);
    const Operand<T> oq(p.q, p.q_st, p.q_sh, p.dim), ok(p.k, p.k_st, p.k_sh, p.dim), ov(p.v, p.v_st, p.v_sh, p.dim);
    const float c2 = p.scale * kLog2e;

    if (tid == 0) {
        tc::mbar_init(bar_s, 1);
        tc::mbar_init(bar_o, 1);
        tc::mbar_init_fence();
    }
    if (warp == 0) tc::tmem_alloc<kCols>(tc::smem_addr(slot_tmem));
    for (int e = tid; e < entries * p.pack; e += kRows) E[e] = bias_entry(p.bias, p.heads, head0 + e / entries, e % entries);
    tc::fence_before();
    __syncthreads();
    tc::fence_after();
    const uint32_t tmem = *slot_tmem, lane_at = static_cast<uint32_t>(warp * 32) << 16;
    const uint32_t ts = tmem + lane_at, to = ts + KT;
    const uint32_t id_o = tc::idesc(kBf16, dim16, false, true);
    int par_s = 0, par_o = 0;  // parities of the next wait
    bool alive = true;

    for (int it = blockIdx.x; it < slots; it += gridDim.x) {
        AttnTile t;
        // causal windows: the last tiles see the most keys and go first
        if (!attn_tile(p.q_off, p.tq, p.k_off, p.tk, p.windows, p.pack, kRows, p.causal ? slots - 1 - it : it, t)) continue;
        const int rows = min(kRows, t.len * p.pack - t.first);
        const int row = t.first + tid;
        const bool live = tid < rows;
        const int see = !live ? 0 : p.causal ? min(max(row / p.pack + t.olen - t.len + 1, 0), t.olen) : t.olen;
        const int most = p.causal ? min(max((t.first + rows - 1) / p.pack + t.olen - t.len + 1, 0), t.olen) : t.olen;
        const int least = p.causal ? min(max(t.first / p.pack + t.olen - t.len + 1, 0), t.olen) : t.olen;  // of the live rows
        const int tiles = (most + KT - 1) / KT, per = (tiles + p.splits - 1) / p.splits;
        const int tile0 = min(static_cast<int>(blockIdx.z) * per, tiles), tile1 = min(tile0 + per, tiles);
        const int64_t token = t.begin + (live ? row / p.pack : 0);
        const int head = head0 + (live ? row % p.pack : 0);

        float m = -INFINITY, l = 0.0f;  // m: what the weights are taken against
        int2 qp = make_int2(0, 0);
        __syncthreads();  // the last tile's staging has been read
        if (tile0 < tile1) {
            const int k0 = tile0 * KT, n = min(KT, most - k0), n16 = (n + 15) & ~15;
            load_panel<T>(sq, kRows, oq, t.begin, head0, p.pack, t.first, rows, kRows, p.dim);
            load_panel<T>(sk, KT, ok, t.obegin + k0, kvh, 1, 0, n, n16, p.dim);
            tc::cp_async_commit();
            load_panel<T>(sv, KT, ov, t.obegin + k0, kvh, 1, 0, n, n16, p.dim);
            tc::cp_async_commit();
            if (entries > 0) {
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
                alive = alive && tc::mbar_wait(bar_o, par_o);
                par_o ^= 1;
            }
            if (tid == 0) {
                tc::fence_after();
                tc::mma_nt(tmem, sq, kRows, sk, KT, dim16, tc::idesc(kBf16, n16, false, false));
                tc::commit(bar_s);
            }
            if (kt > tile0) {
                load_panel<T>(sv, KT, ov, t.obegin + k0, kvh, 1, 0, n, n16, p.dim);
                tc::cp_async_commit();
            }
            BiasMode mode = kOne;
            if (entries > 0) mode = bias_mode(p.bias, join(join(qrange[0], qrange[1]), join(qrange[2], qrange[3])), key_range(kp));
            alive = alive && tc::mbar_wait(bar_s, par_s);
            par_s ^= 1;
            tc::fence_after();
            if (kt + 1 < tile1) {
                const int n2 = min(KT, most - k0 - KT);
                load_panel<T>(sk, KT, ok, t.obegin + k0 + KT, kvh, 1, 0, n2, (n2 + 15) & ~15, p.dim);
            }
            tc::cp_async_commit();  // a group for each tile, an empty one after the last

            // the row's scores, in base 2
            float s[KT];
#pragma unroll
            for (int c = 0; c < KT; c += 16)
                if (c < n16) tc::tmem_ld16(ts + c, s + c);
            tc::wait_ld();
            const bool whole = n == n16 && k0 + n <= least;  // rows past the last one come to nothing anyway
            float top = -INFINITY;
#pragma unroll
            for (int c = 0; c < KT; c += 16) {
                if (c >= n16) continue;
                float(&x)[16] = *reinterpret_cast<float(*)[16]>(s + c);
                if (entries > 0) {
                    add_bias<KT, 16>(x, c2, p.bias, mode, E + (live ? row % p.pack : 0) * entries, kp, c, qp);
                } else {
#pragma unroll
                    for (int i = 0; i < 16; ++i) x[i] *= c2;
                }
                if (!whole) {
#pragma unroll
                    for (int i = 0; i < 16; ++i) x[i] = k0 + c + i < see ? x[i] : -INFINITY;
                }
#pragma unroll
                for (int i = 0; i < 16; ++i) top = fmaxf(top, x[i]);
            }
            // fmaxf passes NaN scores by: their weights are NaN whatever m is, and so is the row
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
            const float off = m == -INFINITY ? 0.0f : m;
            float sum0 = 0.0f, sum1 = 0.0f;
#pragma unroll
            for (int c = 0; c < KT; c += 16) {
                if (c >= n16) continue;
                uint32_t w[8];
#pragma unroll
                for (int i = 0; i < 16; i += 2) {
                    const float a = ex2(s[c + i] - off), b = ex2(s[c + i + 1] - off);
                    sum0 += a;
                    sum1 += b;
                    w[i / 2] = pack2(a, b, T{});
                }
                tc::tmem_st8(ts + c / 2, w);
            }
            l = l * keep + (sum0 + sum1);
            tc::wait_st();
            tc::cp_async_wait<1>();  // V of this tile
            tc::fence_async();
            tc::fence_before();
            __syncthreads();
            if (tid == 0) {
                tc::fence_after();
                tc::mma_tn(tmem + KT, tmem, sv, KT, n16, id_o, kt > tile0);
                tc::commit(bar_o);
            }
            if (entries > 0 && kt + 1 < tile1) load_key_pos<KT>(kp, p.bias, t.obegin + k0 + KT, min(KT, most - k0 - KT));
        }
        if (tile0 < tile1) {
            alive = alive && tc::mbar_wait(bar_o, par_o);
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
            for (int i = 0; i < 16; ++i) fine = fine && is_finite(o[i]);  // columns past dim are 0
            if (p.splits > 1) {
                if (live) write_part(p.part_o + part * p.dim, o, c, p.dim);
            } else {
                stage16<T>(sq, tid, o, c, alive ? inv : __uint_as_float(0x7fffffffu));
            }
        }
        if (p.causal && live && !fine) {
            forward_row<T>(p, token, head, entries > 0 ? p.bias.k_pos : nullptr, t.obegin, tile0 * KT, min(see, tile1 * KT),
                           m == -INFINITY ? 0.0f : m, E + (row % p.pack) * entries, qp, sq,
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

template <typename T, int KT, int DP>
cudaError_t fwd_one(const AttnParams& p, cudaStream_t s) {
    using L = FwdSmem<KT, DP>;
    const int entries = bias_entries(p.bias);
    const int bytes = 1024 + L::kBytes + 4 * entries * p.pack;
    cudaError_t err = cudaFuncSetAttribute(k_attn_fwd_mma<T, KT, DP>, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (err != cudaSuccess) return err;
    // Blocks stay for several tiles of one head; four rounds of them even out tiles of unequal
    // length, one where each has to expand a bias first.
    const int groups = p.heads / p.pack, resident = 148 * (KT == 64 ? 4 : 2) * (entries > 0 ? 1 : 4);
    const int slots = attn_slots(static_cast<int64_t>(p.tq) * p.pack, p.windows, kRows);
    const int per_head = (resident + groups * p.splits - 1) / (groups * p.splits);
    k_attn_fwd_mma<T, KT, DP><<<dim3(slots < per_head ? slots : per_head, groups, p.splits), kRows, bytes, s>>>(p);
    return cudaGetLastError();
}

}  // namespace

cudaError_t launch_attn_forward_mma(const AttnParams& p, int type, cudaStream_t s) {
    if (type == kBF16) return p.dim <= 64 ? fwd_one<__nv_bfloat16, 64, 64>(p, s) : fwd_one<__nv_bfloat16, 128, 128>(p, s);
    return p.dim <= 64 ? fwd_one<__half, 64, 64>(p, s) : fwd_one<__half, 128, 128>(p, s);
}

cudaError_t attn_timeouts(unsigned int* count) {
    return cudaMemcpyFromSymbol(count, g_timeouts, sizeof(unsigned int));
}

}  // namespace oss
