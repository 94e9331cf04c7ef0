// Attention of new tokens over a paged cache, many rows: prompts and long chunks on tcgen05.
//
// A block owns 256 rows (token, query head of the group) of one (sequence, cached head) as two
// tiles of 128 and streams the keys and values that they see in tiles of 128, so that a tile in
// shared memory serves both row tiles. Warps 0-3 and 4-7 hold the two row tiles, a thread a row
// (TMEM lane); warp 8 issues the MMAs, warp 9 the TMA loads, one per page that a tile touches.
// TMEM (512 columns): the scores S of each row tile (128 columns), which its f16 probabilities
// overwrite (two keys a column), and its weighted values O. The MMAs of one row tile run while
// the other's softmax does: per key tile, in the order of issue and so of execution,
//   O0 += P0 V_j, S0 = Q0 K_{j+1}, O1 += P1 V_j, S1 = Q1 K_{j+1}.
// (A warp for each row tile's MMAs let them mix, so that both softmaxes waited and ran together:
// 1.17 -> 1.36 ms for 2048 tokens of 32 heads over 34,816 keys.)
// A commit covers every earlier MMA, so a full S_{j+1} also says that O holds tile j: the softmax
// may rescale it. It does so only when a row's maximum passes its reference by more than 2^8
// (probabilities then lie in (0, 2^8], in f16 lifted by kLift to (0, 2^15]).
#include "paged.cuh"

#include <algorithm>
#include <climits>

namespace tsb {

int device_sm_count();

namespace {

constexpr int PT_THREADS = 384;         // two softmax warpgroups; MMA, TMA and two idle warps
// The softmax warpgroups take registers from the third: 2 * 128 * 216 + 128 * 72 = 384 * 168, what
// the block is launched with.
constexpr int PT_LAUNCH_REGS = 168, PT_SOFTMAX_REGS = 216, PT_OTHER_REGS = 72;
static_assert(256 * PT_SOFTMAX_REGS + 128 * PT_OTHER_REGS <= PT_THREADS * PT_LAUNCH_REGS);
constexpr int PT_KT = 128;
constexpr uint32_t PT_TMEM = 512, PT_O_COL = 256;
constexpr float PT_RESCALE = 8.f;       // log2 of the largest probability kept unscaled

template <int HD>
struct TilesLayout {
    static constexpr int HALF = 128 * 128;                       // 128 rows of 64 values
    static constexpr int SLOT = HD / 64 * HALF;                  // a key tile, a value tile or a row tile
    static constexpr int STAGES = HD == 64 ? 8 : 5;
    static constexpr int SMEM = 1024 + (2 + STAGES) * SLOT + 256;
};

struct TilesBars {
    uint64_t full[8], empty[8], q_ready[2], s_full[2], p_ready[2][2], o_full[2], done;
    uint32_t tmem;
    int abort;
};
static_assert(sizeof(TilesBars) <= 256);

// Bounded waits of this kernel's roles. No suspend-time hint: a warp that sleeps on one wakes some
// hundred cycles late, which stands between every two steps here (1.19 -> 1.09 ms for 2048 tokens of
// 32 heads over 34,816 keys).
__device__ __forceinline__ bool try_wait(uint64_t* bar, uint32_t parity) {
    uint32_t ok;
    asm volatile(
        "{\n .reg .pred p;\n mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n selp.u32 %0, 1, 0, p;\n}\n"
        : "=r"(ok)
        : "r"(smem_u32(bar)), "r"(parity)
        : "memory");
    return ok != 0;
}
__device__ __forceinline__ bool role_wait(uint64_t* bar, uint32_t parity, volatile int* abort, int* err) {
    if (try_wait(bar, parity)) return true;
    const long long start = clock64();
    while (true) {
        if (try_wait(bar, parity)) return true;
        if (*abort) return false;
        if (clock64() - start > kWaitCycles) { *abort = 1; record_error(err, kDevTimeoutAttn); return false; }
    }
}
// Every lane waits; the warp goes on together.
__device__ __forceinline__ bool role_wait_warp(uint64_t* bar, uint32_t parity, volatile int* abort, int* err) {
    const bool ok = role_wait(bar, parity, abort, err);
    return __all_sync(0xffffffffu, ok);
}

__device__ __forceinline__ uint64_t desc_of(uint32_t lo, uint32_t hi) {
    uint64_t d;
    asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "r"(lo), "r"(hi));
    return d;
}
// Two f32 values in a register pair, for the instructions that work on both at once.
using F2 = unsigned long long;
__device__ __forceinline__ F2 f2(float a, float b) {
    F2 r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ void f2_split(F2 x, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(x)); }
__device__ __forceinline__ F2 f2_add(F2 a, F2 b) {
    F2 r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ F2 f2_fma(F2 a, F2 b, F2 c) {
    F2 r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
// MMAs and commits of a converged warp, issued by its elected lane: with the warp together the
// descriptors stay in uniform registers, where a branch for one lane moves them there for each MMA.
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool accumulate) {
    asm volatile(
        "{\n .reg .pred p, e;\n setp.ne.b32 p, %4, 0;\n elect.sync _|e, 0xffffffff;\n"
        " @e tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}\n" ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(uint32_t(accumulate))
        : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, bool accumulate) {
    asm volatile(
        "{\n .reg .pred p, e;\n setp.ne.b32 p, %4, 0;\n elect.sync _|e, 0xffffffff;\n"
        " @e tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}\n" ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"(uint32_t(accumulate))
        : "memory");
}
__device__ __forceinline__ void mma_commit_warp(uint64_t* bar) {
    asm volatile(
        "{\n .reg .pred e;\n elect.sync _|e, 0xffffffff;\n"
        " @e tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n}\n" ::"r"(smem_u32(bar))
        : "memory");
}

template <class T, int HD>
__global__ void __launch_bounds__(PT_THREADS, 1)
    paged_tiles_kernel(const __grid_constant__ PageMaps maps, const PagedAttention a, const PagedGrid grid) {
    using L = TilesLayout<HD>;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* qbuf = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint8_t* ring = qbuf + 2 * L::SLOT;
    TilesBars* bars = reinterpret_cast<TilesBars*>(ring + L::STAGES * L::SLOT);
    volatile int* abort = &bars->abort;
    const int warp = __shfl_sync(0xffffffffu, threadIdx.x / 32, 0), lane = threadIdx.x % 32;    // (known to be uniform)

    uint32_t split;
    int splits;
    const uint32_t item = unit_of(grid, blockIdx.x, &split, &splits);
    const PagedItem it = item_of(grid, item);
    const int m0 = it.row_tile * kPagedTileRows, kvh = it.kvh, seq = it.seq;
    const SeqInfo q = load_seq(a.batch, seq, a.err);
    const int rows = min(kPagedTileRows, q.n * a.group - m0);
    if (rows <= 0) return;
    const int base = q.len - q.n;
    auto position = [&](int r) { return base + int(grid.group.div(m0 + r)); };
    const int hi = position(rows - 1) + 1;
    const int lo = a.window ? max(0, position(0) - a.window + 1) : 0;
    const int tile0 = lo / PT_KT, tiles = (hi + PT_KT - 1) / PT_KT - tile0;
    const int share = splits > 1 ? int(grid.splits.div(tiles + splits - 1)) : tiles;
    const int first = tile0 + int(split) * share, n = min(share, tile0 + tiles - first);
    // key tiles of each row tile in this block's share
    int ng[2];
#pragma unroll
    for (int g = 0; g < 2; ++g) {
        const int last_row = min(rows, (g + 1) * 128) - 1;
        ng[g] = last_row < g * 128 || n <= 0 ? 0 : min(n, max(0, (position(last_row) + PT_KT) / PT_KT - first));
    }
    const int nt = max(ng[0], ng[1]);

    const int t = threadIdx.x & 127, g = threadIdx.x >> 7;         // (warps 0-7)
    const int row = g * 128 + t;
    const bool live = warp < 8 && row < rows;
    uint32_t in_group;
    const int64_t token = q.start + int64_t(grid.group.divmod(m0 + row, &in_group));
    const int head = kvh * a.group + int(in_group);
    const int64_t part = (int64_t(item - grid.whole) * splits + split) * kPagedTileRows + row;
    if (nt == 0) {                                                  // (only with splits)
        if (live) a.part_ml[part] = make_float2(-INFINITY, 0.f);
        return;
    }

    if (threadIdx.x == 0) {
        for (int s = 0; s < L::STAGES; ++s) { mbar_init(&bars->full[s], 1); mbar_init(&bars->empty[s], 1); }
        for (int i = 0; i < 2; ++i) {
            mbar_init(&bars->q_ready[i], 4); mbar_init(&bars->s_full[i], 1);
            mbar_init(&bars->p_ready[i][0], 4); mbar_init(&bars->p_ready[i][1], 4); mbar_init(&bars->o_full[i], 1);
        }
        mbar_init(&bars->done, 1);
        bars->abort = 0;
        mbar_fence_init();
        fence_proxy_async();
    }
    if (warp == 8) { tmem_alloc(&bars->tmem, PT_TMEM); tmem_relinquish(); }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tbase = bars->tmem;

    if (warp >= 8) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(PT_OTHER_REGS));
        if (warp == 9) {
            // TMA producer: K_0, V_0, K_1, V_1, ... through one ring; lane p loads page piece p of a tile.
            const int slots = 1 << a.cache.page_shift, box = min(slots, PT_KT);
            const int* table = a.cache.table + int64_t(seq) * a.cache.table_stride;
            const int key0 = first * PT_KT + lane * box;
            auto page_of = [&](int j) {
                const int key = key0 + j * PT_KT;
                if (lane * box >= PT_KT || j >= nt || key + box <= lo || key >= hi) return -1;
                const int page = table[key >> a.cache.page_shift];
                if (page >= 0 && page < a.cache.num_pages) return page;
                if (any_valid(a, seq, base, max(key, lo), min(key + box, hi))) record_error(a.err, kDevBadPage);
                return a.cache.num_pages;                              // outside the map: zeros
            };
            int next = page_of(0), page = -1;
            int i = 0;
            for (; i < 2 * nt; ++i) {
                const int j = i >> 1, s = i % L::STAGES;
                if ((i & 1) == 0) { page = next; next = page_of(j + 1); }
                if (i >= L::STAGES && !role_wait_warp(&bars->empty[s], ((i / L::STAGES) - 1) & 1, abort, a.err)) break;
                const int pieces = __popc(__ballot_sync(0xffffffffu, page >= 0));
                if (lane == 0) mbar_arrive_expect_tx(&bars->full[s], pieces * box * HD * 2);
                __syncwarp();
                if (page >= 0) {
                    const int slot = (key0 + j * PT_KT) & (slots - 1);
                    uint8_t* dst = ring + s * L::SLOT + lane * box * 128;
#pragma unroll
                    for (int h = 0; h < HD / 64; ++h)
                        load_page(dst + h * L::HALF, (i & 1) ? maps.v : maps.k, &bars->full[s], h * 64, slot, kvh, page);
                }
                __syncwarp();
            }
            // every load has landed before the block ends, also where an abort ends it
            const int from = max(0, i - L::STAGES);
            if (lane == 0) drain(bars->full, L::STAGES, from % L::STAGES, (from / L::STAGES) & 1, i - from);
            __syncwarp();
        } else if (warp == 8) {
            {
                // Few instructions between the MMAs, which they would hold up: descriptors differ from the ring
                // slot's in their low word alone, by constants.
                constexpr uint32_t bf = std::is_same<T, __nv_bfloat16>::value ? kIdescBf16 : 0u;
                const uint32_t id_qk = idesc_f16(128, PT_KT) | bf, id_pv = idesc_f16_bmn(128, HD) | bf;
                const uint64_t dq = smem_desc_sw128(smem_u32(qbuf)), dr = smem_desc_sw128(smem_u32(ring));
                const uint64_t dv = smem_desc_sw128_mn(smem_u32(ring), L::HALF);
                const uint32_t hi = uint32_t(dq >> 32), hi_v = uint32_t(dv >> 32), lo_q = uint32_t(dq), lo_r = uint32_t(dr), lo_v = uint32_t(dv);
                constexpr uint32_t SLOT16 = L::SLOT >> 4;
                int slot = 0, phase = 0;                                // of the next tile in the ring
                auto full = [&]() { return role_wait_warp(&bars->full[slot], phase, abort, a.err); };
                auto next = [&]() { if (++slot == L::STAGES) { slot = 0; phase ^= 1; } };
                auto scores = [&](int gg) {                             // S_gg = Q_gg K of the ring's next tile
                    const uint32_t q = lo_q + gg * SLOT16, k = lo_r + slot * SLOT16;
#pragma unroll
                    for (int i = 0; i < HD / 16; ++i) {
                        const uint32_t off = (i / 4) * (L::HALF >> 4) + (i % 4) * 2;
                        mma_ss(tbase + gg * 128, desc_of(q + off, hi), desc_of(k + off, hi), id_qk, i > 0);
                    }
                    mma_commit_warp(&bars->s_full[gg]);
                };
                bool ok = full();
#pragma unroll
                for (int gg = 0; gg < 2; ++gg)
                    if (ok && ng[gg] > 0) {
                        ok = role_wait_warp(&bars->q_ready[gg], 0, abort, a.err);
                        tc_fence_after();
                        if (ok) scores(gg);
                    }
                if (ok) mma_commit_warp(&bars->empty[0]);
                next();
                for (int j = 0; j < nt && ok; ++j) {
                    ok = full();
                    const int vslot = slot;
                    const uint32_t v = lo_v + slot * SLOT16;
                    next();
                    if (ok && j + 1 < nt) ok = full();
#pragma unroll
                    for (int gg = 0; gg < 2; ++gg) {
                        if (ok && j < ng[gg]) {
                            // the first half of the probabilities is multiplied while the second is made
#pragma unroll
                            for (int h = 0; h < 2; ++h) {
                                if (ok) ok = role_wait_warp(&bars->p_ready[gg][h], j & 1, abort, a.err);
                                tc_fence_after();
                                if (!ok) break;
#pragma unroll
                                for (int kk = 4 * h; kk < 4 * h + 4; ++kk)
                                    mma_ts(tbase + PT_O_COL + gg * 128, tbase + gg * 128 + kk * 8, desc_of(v + kk * 128, hi_v), id_pv,
                                               j > 0 || kk > 0);
                            }
                            if (ok && j + 1 < ng[gg]) scores(gg);
                            if (ok && j + 1 == ng[gg]) mma_commit_warp(&bars->o_full[gg]);
                        }
                        if (ok && gg == 1) mma_commit_warp(&bars->empty[vslot]);
                    }
                    if (ok && j + 1 < nt) { mma_commit_warp(&bars->empty[slot]); next(); }
                }
            }
            // no MMA or commit is left when the block ends and its tensor memory is freed
            mma_commit_warp(&bars->done);
            if (lane == 0) drain(&bars->done, 1, 0, 0, 1);
            __syncwarp();
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(PT_SOFTMAX_REGS));
        // Softmax of row `row`, a thread of TMEM lane t.
        const int ngg = g ? ng[1] : ng[0];
        const uint32_t lanes = uint32_t((warp & 3) * 32) << 16;
        const uint32_t ts = tbase + lanes + g * 128, to = tbase + lanes + PT_O_COL + g * 128;
        const int pos = live ? position(row) : -1;
        const int rows_g = min(rows - g * 128, 128);
        const int pos_first = position(g * 128), pos_last = rows_g > 0 ? position(g * 128 + rows_g - 1) : -1;
        const int from = a.window ? pos - a.window + 1 : 0;         // the row sees positions from .. pos
        const float scale = fabsf(a.scale_log2);
        if (ngg > 0) {
            // the row tile goes to shared memory by its threads (any strides); with a negative scale its
            // signs turn, so that the largest product has the largest score
            const uint32_t flip = a.scale_log2 < 0.f ? 0x80008000u : 0u;
            const uint4* src = reinterpret_cast<const uint4*>(static_cast<const T*>(a.q.data) + token * a.q.token + head * a.q.head);
#pragma unroll
            for (int c = 0; c < HD / 8; ++c) {
                uint4 u = live ? src[c] : make_uint4(0, 0, 0, 0);
                u.x ^= flip; u.y ^= flip; u.z ^= flip; u.w ^= flip;
                *reinterpret_cast<uint4*>(qbuf + g * L::SLOT + (c / 8) * L::HALF + t * 128 + (((c & 7) ^ (t & 7)) << 4)) = u;
            }
            fence_proxy_async();
            __syncwarp();
            if (lane == 0) mbar_arrive(&bars->q_ready[g]);
        }
        // Tiles [plain_from, plain_to) of this block's share are seen whole by every row of the row tile.
        const int plain_to = a.key_valid ? 0 : (pos_first + 1) / PT_KT - first;
        const int plain_from = a.window && pos_last >= a.window ? (pos_last - a.window) / PT_KT + 1 - first : 0;
        const F2 scale2 = f2(scale, scale);
        float mref = -INFINITY;
        F2 acc[4] = {f2(0.f, 0.f), f2(0.f, 0.f), f2(0.f, 0.f), f2(0.f, 0.f)};       // the row's sum, in eight parts
        bool ok = true;
        for (int j = 0; j < ngg; ++j) {
            const bool plain = j >= plain_from && j < plain_to;
            const int k0 = (first + j) * PT_KT;
            uint32_t vw[4] = {~0u, ~0u, ~0u, ~0u};
            if (__builtin_expect(!plain, 0)) {
                if (a.key_valid)
#pragma unroll
                    for (int w = 0; w < 4; ++w) vw[w] = valid_word(a, seq, k0 + w * 32);
                const bool dead_keys = k0 < lo || k0 + PT_KT > hi || (vw[0] & vw[1] & vw[2] & vw[3]) != ~0u;
                if (dead_keys && g == (j < ng[0] ? 0 : 1)) {
                    // values of keys that no row of the block sees: zeros instead of what stands there
                    const int i = 2 * j + 1;
                    if (!(ok = role_wait_warp(&bars->full[i % L::STAGES], (i / L::STAGES) & 1, abort, a.err))) break;
                    const int key = k0 + t;
                    const uint32_t word = t < 64 ? (t < 32 ? vw[0] : vw[1]) : (t < 96 ? vw[2] : vw[3]);
                    const bool valid = ((word >> lane) & 1) || (a.self_visible && key >= base);
                    if (key < lo || key >= hi || !valid) {
                        uint8_t* v = ring + i % L::STAGES * L::SLOT + t * 128;
#pragma unroll
                        for (int h = 0; h < HD / 64; ++h)
#pragma unroll
                            for (int c = 0; c < 8; ++c) *reinterpret_cast<uint4*>(v + h * L::HALF + (((c + t) & 7) << 4)) = make_uint4(0, 0, 0, 0);
                    }
                    fence_proxy_async();
                }
            }
            if (!(ok = role_wait_warp(&bars->s_full[g], j & 1, abort, a.err))) break;
            tc_fence_after();
            // The reference of the earlier tiles serves this one too unless the maximum passes it by more
            // than 2^8, so the first half of the probabilities is made with it while the scores come in, a
            // quarter at a time, and made again in the rare other case.
            uint32_t s[4][32], pk[32];
            float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
            F2 off2;
            auto reference = [&]() {
                const float off = mref == -INFINITY ? 0.f : kLift<T> - mref;
                off2 = f2(off, off);
            };
            auto quarter = [&](const uint32_t (&x)[32], uint32_t* to16) {
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    const F2 y = f2_fma(f2(__uint_as_float(x[2 * e]), __uint_as_float(x[2 * e + 1])), scale2, off2);
                    float e0, e1;
                    f2_split(y, e0, e1);
                    e0 = exp2_ftz(e0);
                    e1 = exp2_ftz(e1);
                    acc[e & 3] = f2_add(acc[e & 3], f2(e0, e1));
                    to16[e] = Pair<T>::down(e0, e1);
                }
            };
            auto hand_over = [&](int half) {
                tmem_st_wait();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&bars->p_ready[g][half]);
            };
            auto maximum = [&](const uint32_t (&x)[32]) {
#pragma unroll
                for (int e = 0; e < 32; e += 2)
                    mx[(e / 2) & 3] = fmaxf(fmaxf(mx[(e / 2) & 3], __uint_as_float(x[e])), __uint_as_float(x[e + 1]));
            };
            tmem_ld32(ts, s[0]);
            // (the common way is laid out in one run: a jump costs a fetch from far behind the instruction cache)
            if (__builtin_expect(plain, 1)) {
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    tmem_ld_wait32(s[c]);
                    if (c < 3) tmem_ld32(ts + (c + 1) * 32, s[c + 1]);
                    maximum(s[c]);
                }
            } else {
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    tmem_ld_wait32(s[c]);
                    if (c < 3) tmem_ld32(ts + (c + 1) * 32, s[c + 1]);
                    const int w0 = k0 + c * 32;
                    const uint32_t see = (vw[c] & range32(from, pos, w0)) | (a.self_visible ? range32(pos, pos, w0) : 0u);
#pragma unroll
                    for (int e = 0; e < 32; ++e)
                        if (!((see >> e) & 1u)) s[c][e] = __float_as_uint(-INFINITY);
                    maximum(s[c]);
                }
            }
            const float mt = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * scale;
            const bool need = mt > mref + PT_RESCALE;                  // (and where nothing was seen before)
            if (__builtin_expect(__any_sync(0xffffffffu, need), 0)) {
                const float factor = need ? exp2_ftz(mref - mt) : 1.f;
                if (need) mref = mt;
                const F2 f = f2(factor, factor), zero = f2(0.f, 0.f);
#pragma unroll
                for (int i = 0; i < 4; ++i) acc[i] = f2_fma(acc[i], f, zero);
                if (j > 0) {
#pragma unroll 1
                    for (int c0 = 0; c0 < HD; c0 += 32) {
                        uint32_t o[32];
                        tmem_ld32(to + c0, o);
                        tmem_ld_wait();
#pragma unroll
                        for (int c = 0; c < 32; ++c) o[c] = __float_as_uint(__uint_as_float(o[c]) * factor);
                        tmem_st32(to + c0, o);
                    }
                }
            }
            reference();
            quarter(s[0], pk);
            quarter(s[1], pk + 16);
            tmem_st32(ts, pk);
            quarter(s[2], reinterpret_cast<uint32_t*>(s[0]));
            hand_over(0);
            quarter(s[3], reinterpret_cast<uint32_t*>(s[0]) + 16);
            tmem_st32(ts + 32, s[0]);
            hand_over(1);
        }
        float sum;
        {
            float s0, s1;
            f2_split(f2_add(f2_add(acc[0], acc[1]), f2_add(acc[2], acc[3])), s0, s1);
            sum = s0 + s1;
        }
        if (ok && ngg > 0) ok = role_wait_warp(&bars->o_full[g], 0, abort, a.err);
        if (ok) {
            tc_fence_after();
            const bool none = ngg == 0;
            if (splits > 1 && live) a.part_ml[part] = none ? make_float2(-INFINITY, 0.f) : make_float2(mref, sum);
            const float inv = none || mref == -INFINITY ? 0.f : splits > 1 ? 1.f : 1.0f / sum;
            const T* gate = a.gate.data ? static_cast<const T*>(a.gate.data) + token * a.gate.token + head * a.gate.head : nullptr;
            T* out = static_cast<T*>(a.out.data) + token * a.out.token + head * a.out.head;
#pragma unroll 1
            for (int c0 = 0; c0 < HD; c0 += 32) {
                uint32_t o[32];
                if (none) {
#pragma unroll
                    for (int c = 0; c < 32; ++c) o[c] = 0u;
                } else {
                    tmem_ld32(to + c0, o);
                    tmem_ld_wait();
                }
                if (!live) continue;
                if (splits > 1) {
                    if (none) continue;
                    float4* dst = reinterpret_cast<float4*>(a.part_o + part * HD + c0);
#pragma unroll
                    for (int c = 0; c < 8; ++c)
                        dst[c] = make_float4(__uint_as_float(o[4 * c]), __uint_as_float(o[4 * c + 1]), __uint_as_float(o[4 * c + 2]),
                                             __uint_as_float(o[4 * c + 3]));
                    continue;
                }
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    float y[8];
#pragma unroll
                    for (int e = 0; e < 8; ++e) y[e] = __uint_as_float(o[8 * c + e]) * inv;
                    if (gate) {
                        float gt[8];
                        unpack8<T>(*reinterpret_cast<const uint4*>(gate + c0 + 8 * c), gt);
#pragma unroll
                        for (int e = 0; e < 8; ++e) y[e] *= gt[e];
                    }
                    *reinterpret_cast<uint4*>(out + c0 + 8 * c) = pack8<T>(y);
                }
            }
        }
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (warp == 8) tmem_dealloc(tbase, PT_TMEM);
}

template <class T, int HD>
cudaError_t launch_tiles(const PagedAttention& a, const PagedGrid& grid, cudaStream_t stream) {
    using L = TilesLayout<HD>;
    const bool bf16 = std::is_same<T, __nv_bfloat16>::value;
    const PagedCache& c = a.cache;
    PageMaps maps;
    if (!page_maps(&maps, c, bf16, PT_KT)) return cudaErrorInvalidValue;
    static KernelSetup configured;
    int dev = 0;
    cudaGetDevice(&dev);
    unsigned long long key = 0;
    if (configured.needed(dev, &key)) {
        const cudaError_t e = cudaFuncSetAttribute(paged_tiles_kernel<T, HD>, cudaFuncAttributeMaxDynamicSharedMemorySize, L::SMEM);
        if (e != cudaSuccess) return e;
        // the register shares above must not exceed what the block is launched with
        cudaFuncAttributes fa;
        const cudaError_t f = cudaFuncGetAttributes(&fa, paged_tiles_kernel<T, HD>);
        if (f != cudaSuccess) return f;
        if (fa.numRegs < PT_LAUNCH_REGS) return cudaErrorLaunchOutOfResources;
        configured.done(dev, key);
    }
    paged_tiles_kernel<T, HD><<<grid.units, PT_THREADS, L::SMEM, stream>>>(maps, a, grid);
    return cudaGetLastError();
}

}  // namespace

cudaError_t paged_attention_tiles(const PagedAttention& a, const PagedGrid& grid, bool bf16, cudaStream_t stream) {
    if (a.cache.head_dim == 64)
        return bf16 ? launch_tiles<__nv_bfloat16, 64>(a, grid, stream) : launch_tiles<__half, 64>(a, grid, stream);
    return bf16 ? launch_tiles<__nv_bfloat16, 128>(a, grid, stream) : launch_tiles<__half, 128>(a, grid, stream);
}

}  // namespace tsb
