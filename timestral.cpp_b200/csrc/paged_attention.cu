// Attention of new tokens over a paged cache (tsb_paged_attention): causal, grouped heads, sliding
// window, key-valid bits, optional gate.
//
// out = gate * sum_j p_j v_j / sum_j p_j with p_j = 2^(t_j - m), t_j = (q . k_j) * scale * log2(e),
// m a running maximum: one pass over the keys that keeps m, the sum and the weighted values in f32. The p_j are
// rounded to the values' type for the second product, whose MMA takes 16-bit operands (their sum is taken before):
// at most half a step of that type relative to each, so of the weighted mean of |v|.
// The rows of one (sequence, cached head) problem are its (token, query head of the group) pairs,
// row = token * group + head, so that a cached key is read once for the whole group.
#include "paged.cuh"

#include <algorithm>
#include <atomic>
#include <climits>

namespace tsb {

bool make_map_4d_16bit(CUtensorMap* map, const void* base, bool bf16, int width, const int64_t (&size)[3],
                       const int64_t (&stride)[3], const int (&box_rows)[3]);
int device_sm_count();

namespace {

// ---------------------------------------------------------------------------------------
// Few rows (single tokens, short chunks) on mma.sync, bound by the bytes of the cache. The products
// are taken transposed, S^T = K Q^T and O^T = V^T P^T: keys and values fill the 16 rows of the MMA
// and the rows of the problem its 8 columns, so that the one to eight rows of a decoded token pad
// to 8, not to 16 (half the MMAs and exponentials) or to the 128 of tcgen05.
// A warp owns 8 * NR rows. RG warps form a team of 8 * NR * RG rows that streams tiles of keys and
// values through a ring of its own; a block's teams work on different problems (short rows:
// nothing to join), or with JOIN on the tiles of one problem in turn, joined through shared
// memory at the end.
// Tiles come by TMA, a load for each page that they touch (a 16-byte cp.async path cost 350
// instructions a tile and ran at 0.57 of the copy rate, a bulk copy for each row, 40 cycles each,
// at 0.27). What stands at keys that no row sees (behind the length, outside the window, the bit
// clear) is masked in the scores, and the values there are overwritten with zeros.
constexpr int PR_THREADS = 128;
constexpr float PR_RESCALE = 8.f;        // log2 of the largest probability kept unscaled

// ONE: the tile holds every key of the problem (no window, max_length <= KT), so there is no ring, and
// the tile takes no more shared memory than max_length rounded up to 16 keys, for more blocks an SM.
template <int HD, int RG, bool ONE>
struct RowsLayout {
    static constexpr int TEAMS = 4 / RG;
    static constexpr int KT = ONE ? 96 : RG == 4 ? 64 : 32; // keys of a tile
    static constexpr int BOX = ONE ? 16 : KT;         // keys of one load at most
    static constexpr int STAGES = ONE ? 1 : 3;
    static constexpr int HALF = KT * 128;                   // 64 values of the tile's keys
    static constexpr int TILE = HD / 64 * HALF;             // bytes of a tile of keys (or values)
    static constexpr int RING = STAGES * 2 * TILE;
    static constexpr int SMEM = 1024 + TEAMS * RING + TEAMS * STAGES * 8;
    static int smem(int keys) { return ONE ? 1024 + TEAMS * (2 * HD / 64 * keys * 128 + 8) : SMEM; }
    static_assert(ONE || SMEM >= 1024 + (4 * 16 + 16 * RG) * (HD * 4 + 8), "the joined rows reuse the rings");
};

template <class T>
__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1);
template <>
__device__ __forceinline__ void mma16816<__half>(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <>
__device__ __forceinline__ void mma16816<__nv_bfloat16>(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void ldsm4(uint32_t addr, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
// An 8 x 8 block of 16-bit values, held by a warp as a fragment, turned over.
__device__ __forceinline__ uint32_t turn8x8(uint32_t x) {
    uint32_t y;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}
__device__ __forceinline__ void ldsm4_t(uint32_t addr, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
// All warps of a team (a warp alone: the warp).
template <int RG>
__device__ __forceinline__ void team_sync(int team) {
    if constexpr (RG == 1) __syncwarp();
    else asm volatile("bar.sync %0, %1;" ::"r"(team + 1), "n"(32 * RG) : "memory");
}

// What a team works on.
struct RowTile {
    int seq, kvh, m0, rows;      // first row and live rows of the tile
    int base;                    // position of the sequence's first new token
    int lo, hi;                  // keys that any row of the tile may see
    int start;                   // first token row
};

// Of a partial result: no key was seen. (Scores that are all NaN leave the maximum where it was, too,
// and a sum that is NaN.)
__device__ __forceinline__ bool saw_nothing(float maximum, float sum) { return maximum == -INFINITY && sum == 0.f; }

// 16 bytes (8) of another block of the cluster, at this block's shared address.
__device__ __forceinline__ float4 peer_load4(const void* mine, uint32_t rank) {
    float4 v;
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(mapa_shared(smem_u32(mine), rank)) : "memory");
    return v;
}
__device__ __forceinline__ float2 peer_load2(const void* mine, uint32_t rank) {
    float2 v;
    asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(mapa_shared(smem_u32(mine), rank)) : "memory");
    return v;
}

// Eight finished values (columns 8 c ..) of a row: normalised, gated, rounded, stored.
template <class T>
__device__ __forceinline__ void store_row(const PagedAttention& a, int64_t token, int head, int c, float (&y)[8], float inv) {
#pragma unroll
    for (int e = 0; e < 8; ++e) y[e] *= inv;
    if (a.gate.data) {
        float g[8];
        unpack8<T>(*reinterpret_cast<const uint4*>(static_cast<const T*>(a.gate.data) + token * a.gate.token + head * a.gate.head + c * 8), g);
#pragma unroll
        for (int e = 0; e < 8; ++e) y[e] *= g[e];
    }
    *reinterpret_cast<uint4*>(static_cast<T*>(a.out.data) + token * a.out.token + head * a.out.head + c * 8) = pack8<T>(y);
}

// Four 32-bit values a lane, one for each of four 8-value columns of a row that the quad shares:
// afterwards lane i of the quad holds all of column i.
__device__ __forceinline__ void quad_transpose(uint32_t (&v)[4]) {
    const int i = threadIdx.x & 3;
    const bool odd = i & 1, high = i & 2;
    // lane i exchanges with i ^ 1, then with i ^ 2
    uint32_t a = __shfl_xor_sync(0xffffffffu, odd ? v[0] : v[1], 1), b = __shfl_xor_sync(0xffffffffu, odd ? v[2] : v[3], 1);
    if (odd) { v[0] = a; v[2] = b; } else { v[1] = a; v[3] = b; }
    a = __shfl_xor_sync(0xffffffffu, high ? v[0] : v[2], 2);
    b = __shfl_xor_sync(0xffffffffu, high ? v[1] : v[3], 2);
    if (high) { v[0] = a; v[1] = b; } else { v[2] = a; v[3] = b; }
}

template <class T, int HD, int RG, int NR, bool JOIN, bool ONE>
__global__ void __launch_bounds__(PR_THREADS, HD == 128 ? 1 : NR == 1 ? 5 : RG == 4 ? 3 : 4)
    paged_rows_kernel(const __grid_constant__ PageMaps maps, const PagedAttention a, const PagedGrid grid) {
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    using L = RowsLayout<HD, RG, ONE>;
    constexpr int KT = L::KT, MK = KT / 16, NW = KT / 32, KS = HD / 16, MD = HD / 16, WR = 8 * NR, MT = WR * RG;
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, rg = warp % RG, team = warp / RG;

    const uint32_t unit = blockIdx.x * (JOIN ? 1 : L::TEAMS) + (JOIN ? 0 : team);
    if (unit >= grid.units) return;
    RowTile t;
    uint32_t split;
    int splits;
    const uint32_t item = unit_of(grid, unit, &split, &splits);
    const PagedItem it = item_of(grid, item);
    t.seq = it.seq;
    t.kvh = it.kvh;
    t.m0 = it.row_tile * MT;
    const SeqInfo q = load_seq(a.batch, t.seq, a.err);
    t.rows = min(MT, q.n * a.group - t.m0);
    if (t.rows <= 0) return;
    t.start = q.start;
    t.base = q.len - q.n;
    const int t_first = int(grid.group.div(t.m0)), t_last = int(grid.group.div(t.m0 + t.rows - 1));
    t.hi = t.base + t_last + 1;
    t.lo = !ONE && a.window ? max(0, t.base + t_first - a.window + 1) : 0;
    // this item's share of the tiles, and of those this team's
    const int tile0 = ONE ? 0 : t.lo / KT, tiles = ONE ? 1 : (t.hi + KT - 1) / KT - tile0;
    const int share = splits > 1 ? int(grid.splits.div(tiles + splits - 1)) : tiles;
    constexpr int STEP = JOIN ? L::TEAMS : 1;
    const int first = ONE ? 0 : tile0 + int(split) * share + (JOIN ? team : 0);
    const int last = ONE ? 1 : min(tile0 + (int(split) + 1) * share, tile0 + tiles);

    const int half = ONE ? int(grid.one_keys) * 128 : L::HALF, tile_bytes = ONE ? HD / 64 * half : L::TILE;
    uint8_t* ring = smem + team * (L::STAGES * 2 * tile_bytes);
    uint64_t* full = reinterpret_cast<uint64_t*>(smem + L::TEAMS * L::STAGES * 2 * tile_bytes) + team * L::STAGES;
    if (rg == 0 && lane == 0) {
        for (int s = 0; s < L::STAGES; ++s) mbar_init(&full[s], 1);
        mbar_fence_init();
        fence_proxy_async();
    }
    team_sync<RG>(team);

    // The team's first warp loads: lane p the p-th page that the tile touches.
    const int slots = 1 << a.cache.page_shift, box = min(slots, L::BOX);
    const int* table = a.cache.table + int64_t(t.seq) * a.cache.table_stride;
    bool strange = false;                                  // an entry named no page
    auto page_of = [&](int tile) {
        const int key = tile * KT + lane * box;
        if (rg != 0 || tile >= last || lane * box >= KT || key + box <= t.lo || key >= t.hi) return -1;
        const int page = table[key >> a.cache.page_shift];
        if (page >= 0 && page < a.cache.num_pages) return page;
        strange = true;
        return a.cache.num_pages;                          // outside the map: zeros
    };
    auto load_tile = [&](int tile, int stage, int page) {
        if (rg != 0) return;
        const int pieces = __popc(__ballot_sync(0xffffffffu, page >= 0));
        if (lane == 0) mbar_arrive_expect_tx(&full[stage], pieces * box * HD * 4);
        __syncwarp();
        if (page >= 0) {
            const int slot = (tile * KT + lane * box) & (slots - 1);
            uint8_t* dst = ring + stage * 2 * tile_bytes + lane * box * 128;
#pragma unroll
            for (int h = 0; h < HD / 64; ++h) {
                load_page(dst + h * half, maps.k, &full[stage], h * 64, slot, t.kvh, page);
                load_page(dst + tile_bytes + h * half, maps.v, &full[stage], h * 64, slot, t.kvh, page);
            }
        }
        __syncwarp();
    };
    int page = page_of(first);
#pragma unroll
    for (int s = 0; s < (ONE ? 1 : L::STAGES - 1); ++s) {
        if (first + s * STEP < last) load_tile(first + s * STEP, s, page);
        if (!ONE) page = page_of(first + (s + 1) * STEP);
    }

    // Fragments: of a query row this lane holds row lane / 4 (+ 8 n), of a score or weighted value the
    // rows 2 (lane % 4) + {0, 1} (+ 8 n); pos: the latter's positions (rows that are not there: before
    // every key).
    int pos[NR][2];
    uint32_t qf[KS][NR][2];
    // with a negative scale the queries' signs turn, so that the largest product has the largest score
    const uint32_t flip = a.scale_log2 < 0.f ? 0x80008000u : 0u;
    const float scale = fabsf(a.scale_log2);
#pragma unroll
    for (int n = 0; n < NR; ++n) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const int r = rg * WR + n * 8 + (lane & 3) * 2 + e;
            pos[n][e] = r < t.rows ? t.base + int(grid.group.div(t.m0 + r)) : -1;
        }
        const int r = rg * WR + n * 8 + lane / 4, m = t.m0 + r, tok = int(grid.group.div(m));
        const uint32_t* p = reinterpret_cast<const uint32_t*>(static_cast<const T*>(a.q.data) + (t.start + tok) * a.q.token +
                                                              (t.kvh * a.group + m - tok * a.group) * a.q.head) + (lane & 3);
#pragma unroll
        for (int k = 0; k < KS; ++k) {
            qf[k][n][0] = r < t.rows ? p[k * 8] ^ flip : 0u;
            qf[k][n][1] = r < t.rows ? p[k * 8 + 4] ^ flip : 0u;
        }
    }
    // A short problem's gate and key bits are on their way while its keys are.
    uint32_t gv[ONE ? NR : 1][ONE ? HD / 8 : 1];
    if constexpr (ONE) {
        if (a.gate.data)
#pragma unroll
            for (int n = 0; n < NR; ++n) {
                const int r = rg * WR + n * 8 + lane / 4, m = t.m0 + r, tok = int(grid.group.div(m));
                const T* gate = static_cast<const T*>(a.gate.data) + (t.start + tok) * a.gate.token + (t.kvh * a.group + m - tok * a.group) * a.gate.head;
#pragma unroll
                for (int b = 0; b < HD / 8; ++b)
                    gv[n][b] = r < t.rows ? *reinterpret_cast<const uint32_t*>(gate + b * 8 + (lane & 3) * 2) : 0u;
            }
    }
    float o[MD][NR][4];
#pragma unroll
    for (int d = 0; d < MD; ++d)
#pragma unroll
        for (int n = 0; n < NR; ++n) o[d][n][0] = o[d][n][1] = o[d][n][2] = o[d][n][3] = 0.f;
    float mx[NR][2], sum[NR][2];
#pragma unroll
    for (int n = 0; n < NR; ++n) { mx[n][0] = mx[n][1] = -INFINITY; sum[n][0] = sum[n][1] = 0.f; }

    int st = 0, phase = 0;
    bool expired = false;       // after an expired wait the warp goes on, without waits or loads, to meet its team's barriers
    for (int tile = first; tile < last; tile += STEP) {
        const int k0 = ONE ? 0 : tile * KT;
        uint32_t valid[NW];
        bool whole = true;                          // every bit is set
#pragma unroll
        for (int w = 0; w < NW; ++w) valid[w] = a.key_valid ? valid_word(a, t.seq, k0 + w * 32) : ~0u;
        if (!expired && __builtin_expect(!__all_sync(0xffffffffu, mbar_wait(&full[st], phase)), 0)) {
            record_error(a.err, kDevTimeoutAttn);
            expired = true;
            if (rg == 0) drain(full, L::STAGES, st, phase, min(ONE ? 1 : L::STAGES - 1, (last - tile + STEP - 1) / STEP));
        }
        uint8_t* const tk = ring + st * 2 * tile_bytes;
#pragma unroll
        for (int w = 0; w < NW; ++w) whole = whole && valid[w] == ~0u;
        if (k0 < t.lo || k0 + KT > t.hi || !whole) {
            // values of keys that no row sees: zeros instead of what stands there
#pragma unroll
            for (int w = 0; w < NW; ++w) {
                if (NW % RG == 0 ? w % RG != rg : rg != 0) continue;       // a warp a word, or the first all of them
                const int r = w * 32 + lane, key = k0 + r;
                if (ONE && r >= int(grid.one_keys)) continue;
                if (key >= t.lo && key < t.hi && (((valid[w] >> lane) & 1) || (a.self_visible && key >= t.base))) continue;
#pragma unroll
                for (int c = 0; c < HD / 8; ++c)
                    *reinterpret_cast<uint4*>(tk + tile_bytes + (c / 8) * half + r * 128 + (((c + lane) & 7) << 4)) = make_uint4(0, 0, 0, 0);
            }
            fence_proxy_async();                    // before a later load into the stage
        }
        team_sync<RG>(team);                        // zeros are written; the stage read last is free
        if constexpr (!ONE) {
            const int nx = tile + (L::STAGES - 1) * STEP, ns = st == 0 ? L::STAGES - 1 : st - 1;
            if (nx < last && !expired) load_tile(nx, ns, page);
            page = page_of(nx + STEP);
        }
        const uint32_t sk = smem_u32(tk), sv = sk + tile_bytes;
        if (++st == L::STAGES) { st = 0; phase ^= 1; }
        float sc[MK][NR][4];
#pragma unroll
        for (int i = 0; i < MK; ++i)
#pragma unroll
            for (int n = 0; n < NR; ++n) sc[i][n][0] = sc[i][n][1] = sc[i][n][2] = sc[i][n][3] = 0.f;
        const uint32_t ka = sk + (lane & 15) * 128, kx = ((lane & 7) ^ (lane >> 4)) << 4;
        // (16 keys behind the last that the rows see cost nothing; the first 16 of a tile are always tried)
        const int here = ONE ? (t.hi - k0 + 15) / 16 : MK;
#pragma unroll
        for (int i = 0; i < MK; ++i) {
            if (ONE && i >= here) break;
#pragma unroll
            for (int k = 0; k < KS; ++k) {
                uint32_t f[4];
                ldsm4(ka + (k / 4) * half + i * 16 * 128 + (kx ^ ((k % 4) << 5)), f);
#pragma unroll
                for (int n = 0; n < NR; ++n) mma16816<T>(sc[i][n], f, qf[k][n][0], qf[k][n][1]);
            }
        }
        // every row of the tile sees every key of it: no per-key masks
        const bool all = k0 + KT - 1 <= t.base + t_first && (a.window == 0 || k0 > t.base + t_last - a.window) && whole;
        if (!all) {
#pragma unroll
            for (int n = 0; n < NR; ++n)
#pragma unroll
                for (int e = 0; e < 2; ++e)
#pragma unroll
                    for (int w = 0; w < NW; ++w) {
                        // bit 8 j of the row's keys of this word, from this lane's first (lane / 4) on
                        const int p = pos[n][e] - k0 - w * 32;                 // the row's own key, counted from the word
                        uint32_t see = p < 0 ? 0u : p >= 31 ? valid[w] : valid[w] & ((2u << p) - 1);
                        if (!ONE && a.window) see &= range32(p - a.window + 1, 31, 0);
                        if (a.self_visible && p >= 0 && p < 32) see |= 1u << p;
                        see >>= lane >> 2;
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            float& x = sc[w * 2 + j / 2][n][2 * (j & 1) + e];
                            if (!((see >> (8 * j)) & 1)) x = -INFINITY;
                        }
                    }
        }
        // The reference maximum of a row moves only when a score passes it by more than 2^8: then the
        // sums are scaled down, which most tiles spare.
        float m[NR][2];
        bool up = false;
#pragma unroll
        for (int n = 0; n < NR; ++n)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                float x = fmaxf(sc[0][n][e], sc[0][n][2 + e]);
#pragma unroll
                for (int i = 1; i < MK; ++i) x = fmaxf(x, fmaxf(sc[i][n][e], sc[i][n][2 + e]));
                x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 4));
                x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 8));
                x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 16)) * scale;
                m[n][e] = x;
                up |= x > mx[n][e] + PR_RESCALE;
            }
        if constexpr (ONE) {
#pragma unroll
            for (int n = 0; n < NR; ++n) { mx[n][0] = m[n][0]; mx[n][1] = m[n][1]; }
        } else if (__any_sync(0xffffffffu, up)) {
#pragma unroll
            for (int n = 0; n < NR; ++n)
#pragma unroll
                for (int e = 0; e < 2; ++e)
                    if (m[n][e] > mx[n][e] + PR_RESCALE) {
                        const float f = exp2_ftz(mx[n][e] - m[n][e]);
                        mx[n][e] = m[n][e];
                        sum[n][e] *= f;
#pragma unroll
                        for (int d = 0; d < MD; ++d) { o[d][n][e] *= f; o[d][n][2 + e] *= f; }
                    }
        }
#pragma unroll
        for (int n = 0; n < NR; ++n)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const float ref = mx[n][e] == -INFINITY ? 0.f : mx[n][e] - kLift<T>;
#pragma unroll
                for (int i = 0; i < MK; ++i) {
                    sc[i][n][e] = exp2_ftz(fmaf(sc[i][n][e], scale, -ref));
                    sc[i][n][2 + e] = exp2_ftz(fmaf(sc[i][n][2 + e], scale, -ref));
                    sum[n][e] += sc[i][n][e] + sc[i][n][2 + e];
                }
            }
        const uint32_t va = sv + ((lane & 7) + ((lane >> 4) << 3)) * 128, vx = ((lane & 7) ^ ((lane >> 3) & 1)) << 4;
#pragma unroll
        for (int i = 0; i < MK; ++i) {
            if (ONE && i >= here) break;
            uint32_t p[NR][2];
#pragma unroll
            for (int n = 0; n < NR; ++n) {
                p[n][0] = turn8x8(Pair<T>::down(sc[i][n][0], sc[i][n][1]));
                p[n][1] = turn8x8(Pair<T>::down(sc[i][n][2], sc[i][n][3]));
            }
#pragma unroll
            for (int d = 0; d < MD; ++d) {
                uint32_t f[4];
                ldsm4_t(va + (d / 4) * half + i * 16 * 128 + (vx ^ ((d % 4) << 5)), f);
#pragma unroll
                for (int n = 0; n < NR; ++n) mma16816<T>(o[d][n], f, p[n][0], p[n][1]);
            }
        }
    }
    // Was one of those pages to be read? (Looked at again here: in page_of it cost the decode batch 1 %.)
    if (__builtin_expect(strange, 0))
#pragma unroll 1
        for (int tile = first; tile < last; tile += STEP) {
            const int key = tile * KT + lane * box, from = max(key, t.lo), to = min(key + box, t.hi);
            const int page = from < to ? table[key >> a.cache.page_shift] : 0;
            if ((page < 0 || page >= a.cache.num_pages) && any_valid(a, t.seq, t.base, from, to)) record_error(a.err, kDevBadPage);
        }
#pragma unroll
    for (int n = 0; n < NR; ++n)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            sum[n][e] += __shfl_xor_sync(0xffffffffu, sum[n][e], 4);
            sum[n][e] += __shfl_xor_sync(0xffffffffu, sum[n][e], 8);
            sum[n][e] += __shfl_xor_sync(0xffffffffu, sum[n][e], 16);
        }
    const int64_t part = (int64_t(item - grid.whole) * splits + split) * MT;      // row 0 of the tile
    auto row_of = [&](int r, int64_t* token, int* head) {
        const int m = t.m0 + r, tok = int(grid.group.div(m));
        *token = t.start + tok;
        *head = t.kvh * a.group + m - tok * a.group;
    };
    if constexpr (!JOIN) {
#pragma unroll
        for (int n = 0; n < NR; ++n) {
            if (splits > 1) {
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    if (pos[n][e] < 0) continue;
                    const int64_t at = part + rg * WR + n * 8 + (lane & 3) * 2 + e;
                    if (lane < 4) a.part_ml[at] = make_float2(mx[n][e], sum[n][e]);
                    if (saw_nothing(mx[n][e], sum[n][e])) continue;
#pragma unroll
                    for (int d = 0; d < MD; ++d) {
                        a.part_o[at * HD + d * 16 + (lane >> 2)] = o[d][n][e];
                        a.part_o[at * HD + d * 16 + 8 + (lane >> 2)] = o[d][n][2 + e];
                    }
                }
                continue;
            }
            // Fragments turn back to rows, 32 columns at a time so that a lane stores 16 bytes; the gate's
            // 16-bit values turn the other way, so that the product is rounded once.
            const int r = rg * WR + n * 8 + (lane >> 2);
            const bool there = r < t.rows;
            int64_t token;
            int head;
            row_of(r, &token, &head);
            const float inv[2] = {mx[n][0] == -INFINITY ? 0.f : 1.0f / sum[n][0], mx[n][1] == -INFINITY ? 0.f : 1.0f / sum[n][1]};
            const T* gate = static_cast<const T*>(a.gate.data) + token * a.gate.token + head * a.gate.head;
            T* out = static_cast<T*>(a.out.data) + token * a.out.token + head * a.out.head;
#pragma unroll
            for (int b = 0; b < HD / 8; b += 4) {
                uint32_t u[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    float x = o[(b + i) / 2][n][((b + i) & 1) * 2] * inv[0], y = o[(b + i) / 2][n][((b + i) & 1) * 2 + 1] * inv[1];
                    if (a.gate.data) {
                        uint32_t g;
                        if constexpr (ONE) g = gv[n][b + i];
                        else g = there ? *reinterpret_cast<const uint32_t*>(gate + (b + i) * 8 + (lane & 3) * 2) : 0u;
                        const float2 gf = Pair<T>::up(turn8x8(g));
                        x *= gf.x;
                        y *= gf.y;
                    }
                    u[i] = turn8x8(Pair<T>::down(x, y));
                }
                quad_transpose(u);
                if (there) *reinterpret_cast<uint4*>(out + (b + (lane & 3)) * 8) = make_uint4(u[0], u[1], u[2], u[3]);
            }
        }
        return;
    }
    // Join the teams through shared memory: per warp WR rows of HD f32 (columns of 8 turned by the
    // row, against bank conflicts), maximum and sum.
    __syncthreads();
    float* so = reinterpret_cast<float*>(smem) + warp * WR * HD;
    float2* sml = reinterpret_cast<float2*>(smem + 4 * WR * HD * 4);
#pragma unroll
    for (int n = 0; n < NR; ++n)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const int r = n * 8 + (lane & 3) * 2 + e, x = (lane & 3) << 3;
#pragma unroll
            for (int d = 0; d < MD; ++d) {
                so[r * HD + ((d * 16) ^ x) + (lane >> 2)] = o[d][n][e];
                so[r * HD + ((d * 16 + 8) ^ x) + (lane >> 2)] = o[d][n][2 + e];
            }
            if (lane < 4) sml[warp * WR + r] = make_float2(mx[n][e], sum[n][e]);
        }
    __syncthreads();
    constexpr int CH = HD / 8;
    float* share_o = reinterpret_cast<float*>(smem) + 4 * WR * HD + 8 * WR;        // behind the warps' rows and sums
    float2* share_ml = reinterpret_cast<float2*>(share_o + MT * HD);
    for (int i = threadIdx.x; i < t.rows * CH; i += PR_THREADS) {
        const int r = i / CH, c = i % CH, g = r / WR, rr = r % WR;
        float m = -INFINITY;
#pragma unroll
        for (int k = 0; k < L::TEAMS; ++k) m = fmaxf(m, sml[(k * RG + g) * WR + rr].x);
        float y[8] = {}, l = 0.f;
#pragma unroll
        for (int k = 0; k < L::TEAMS; ++k) {
            const int w = k * RG + g;
            const float2 ml = sml[w * WR + rr];
            const float f = ml.x == -INFINITY ? 0.f : exp2_ftz(ml.x - m);
            l = fmaf(ml.y, f, l);
            const float* src = reinterpret_cast<const float*>(smem) + w * WR * HD + rr * HD + ((c * 8) ^ (((rr >> 1) & 3) << 3));
#pragma unroll
            for (int e = 0; e < 8; ++e) y[e] = fmaf(src[e], f, y[e]);
        }
        if (splits > 1 && grid.cluster) {
            float4* dst = reinterpret_cast<float4*>(share_o + r * HD + c * 8);
            dst[0] = make_float4(y[0], y[1], y[2], y[3]);
            dst[1] = make_float4(y[4], y[5], y[6], y[7]);
            if (c == 0) share_ml[r] = make_float2(m, l);
            continue;
        }
        if (splits > 1) {
            const int64_t at = part + r;
            if (c == 0) a.part_ml[at] = make_float2(m, l);
            if (!saw_nothing(m, l)) {
                float4* dst = reinterpret_cast<float4*>(a.part_o + at * HD + c * 8);
                dst[0] = make_float4(y[0], y[1], y[2], y[3]);
                dst[1] = make_float4(y[4], y[5], y[6], y[7]);
            }
            continue;
        }
        int64_t token;
        int head;
        row_of(r, &token, &head);
        store_row<T>(a, token, head, c, y, m == -INFINITY ? 0.f : 1.0f / l);
    }
    if (splits > 1 && grid.cluster) {
        // The splits of an item are one cluster: each block finishes its share of the rows from all of them.
        cluster_sync();
        for (int i = int(split) * PR_THREADS + threadIdx.x; i < t.rows * CH; i += splits * PR_THREADS) {
            const int r = i / CH, c = i % CH;
            float m = -INFINITY;
            for (int k = 0; k < splits; ++k) m = fmaxf(m, peer_load2(share_ml + r, k).x);
            float y[8] = {}, l = 0.f;
            for (int k = 0; k < splits; ++k) {
                const float2 ml = peer_load2(share_ml + r, k);
                const float f = ml.x == -INFINITY ? 0.f : exp2_ftz(ml.x - m);
                const float4 u = peer_load4(share_o + r * HD + c * 8, k), w = peer_load4(share_o + r * HD + c * 8 + 4, k);
                const float p[8] = {u.x, u.y, u.z, u.w, w.x, w.y, w.z, w.w};
                l = fmaf(ml.y, f, l);
#pragma unroll
                for (int e = 0; e < 8; ++e) y[e] = fmaf(p[e], f, y[e]);
            }
            int64_t token;
            int head;
            row_of(r, &token, &head);
            store_row<T>(a, token, head, c, y, m == -INFINITY ? 0.f : 1.0f / l);
        }
        cluster_sync();                             // no block leaves while another reads its shared memory
    }
}

__global__ void drain_selftest_kernel(int* err, const uint8_t* src) {
    __shared__ __align__(128) uint8_t buf[2][1024];
    __shared__ uint64_t bars[2];
    for (int i = threadIdx.x; i < 2 * 1024; i += 32) buf[i / 1024][i % 1024] = 0xff;
    if (threadIdx.x == 0) {
        mbar_init(&bars[0], 1);
        mbar_init(&bars[1], 1);
        mbar_fence_init();
        fence_proxy_async();
    }
    __syncwarp();
    auto load = [&](int s, uint32_t expected) {
        mbar_arrive_expect_tx(&bars[s], expected);
        asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(smem_u32(buf[s])),
                     "l"(src), "r"(1024u), "r"(smem_u32(&bars[s])) : "memory");
    };
    if (threadIdx.x == 0) {
        load(1, 1024);                     // a ring of two, from its second stage on
        load(0, 1024);
    }
    __syncwarp();
    bool ok = drain(bars, 2, 1, 0, 1) && drain(bars, 2, 0, 0, 1);
    for (int i = threadIdx.x; i < 2 * 1024; i += 32) ok = ok && buf[i / 1024][i % 1024] == 0;
    ok = __all_sync(0xffffffffu, ok);
    if (threadIdx.x == 0) {
        if (ok) err[1] = 1;
        load(1, 2 * 1024);                 // (of which the second half never comes)
        load(0, 1024);
    }
    __syncwarp();
    if (!__all_sync(0xffffffffu, drain(bars, 2, 1, 1, 2))) record_error(err, kDevTimeoutAttn);
}

// Join the splits of a row: HD / 8 threads hold a partial row, G groups of them share the splits out
// (8 for many splits of few rows, else 2), joined through shared memory.
template <class T, int HD, int G>
__global__ void __launch_bounds__(128) paged_combine_kernel(const PagedAttention a, const PagedGrid grid, int tile_rows) {
    constexpr int CH = HD / 8, ROWS = 128 / (CH * G);
    __shared__ float so[ROWS * G][HD];
    __shared__ float2 sml[ROWS * G];
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int slot = threadIdx.x / CH, c = threadIdx.x % CH, g = slot % G;
    // tile_rows is a power of two
    const uint32_t row = blockIdx.x * ROWS + slot / G, split_item = row >> (31 - __clz(tile_rows)), r = row & (tile_rows - 1);
    const PagedItem it = item_of(grid, min(grid.whole + split_item, grid.items - 1));
    const SeqInfo q = load_seq(a.batch, it.seq, nullptr);
    uint32_t in_group;
    const int m = it.row_tile * tile_rows + int(r);
    const int64_t token = q.start + int64_t(grid.group.divmod(m, &in_group));
    const int head = it.kvh * a.group + int(in_group);
    const bool live = grid.whole + split_item < grid.items && m < q.n * a.group;
    const int64_t at = int64_t(split_item) * a.splits * tile_rows + r, step = tile_rows;
    float top_m = -INFINITY, y[8] = {}, l = 0.f;
    if (live) {
#pragma unroll 4
        for (int s = g; s < a.splits; s += G) {
            const float2 ml = a.part_ml[s * step + at];
            if (saw_nothing(ml.x, ml.y)) continue;    // no partial row was written
            const float4* src = reinterpret_cast<const float4*>(a.part_o + (s * step + at) * HD + c * 8);
            const float4 u = src[0], w = src[1];
            const float top = fmaxf(top_m, ml.x), f = exp2_ftz(ml.x - top), old = exp2_ftz(top_m - top);
            top_m = top;
            l = fmaf(l, old, ml.y * f);
            const float p[8] = {u.x, u.y, u.z, u.w, w.x, w.y, w.z, w.w};
#pragma unroll
            for (int e = 0; e < 8; ++e) y[e] = fmaf(y[e], old, p[e] * f);
        }
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) so[slot][c * 8 + e] = y[e];
    if (c == 0) sml[slot] = make_float2(top_m, l);
    __syncthreads();
    if (g != 0 || !live) return;
    float top = -INFINITY;
#pragma unroll
    for (int k = 0; k < G; ++k) top = fmaxf(top, sml[slot + k].x);
    l = 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) y[e] = 0.f;
#pragma unroll
    for (int k = 0; k < G; ++k) {
        const float2 ml = sml[slot + k];
        if (saw_nothing(ml.x, ml.y)) continue;
        const float f = exp2_ftz(ml.x - top);
        l = fmaf(ml.y, f, l);
#pragma unroll
        for (int e = 0; e < 8; ++e) y[e] = fmaf(so[slot + k][c * 8 + e], f, y[e]);
    }
    store_row<T>(a, token, head, c, y, top == -INFINITY ? 0.f : 1.0f / l);
}

// Rows of a problem -> warps of a team and their rows: 8, 16, 32 or 64 rows.
int rows_of_team(const PagedAttention& a) {
    const int64_t rows = int64_t(a.batch.max_chunk) * a.group;
    return rows <= 8 ? 8 : rows <= 16 ? 16 : rows <= 32 ? 32 : 64;
}

template <class T, int HD, int RG, int NR, bool JOIN, bool ONE>
cudaError_t launch_rows(const PagedAttention& a, const PagedGrid& grid, cudaStream_t stream) {
    using L = RowsLayout<HD, RG, ONE>;
    static KernelSetup configured;
    int dev = 0;
    cudaGetDevice(&dev);
    unsigned long long key = 0;
    if (configured.needed(dev, &key)) {
        const cudaError_t e = cudaFuncSetAttribute(paged_rows_kernel<T, HD, RG, NR, JOIN, ONE>, cudaFuncAttributeMaxDynamicSharedMemorySize, L::SMEM);
        if (e != cudaSuccess) return e;
        configured.done(dev, key);
    }
    PageMaps maps;
    if (!page_maps(&maps, a.cache, std::is_same<T, __nv_bfloat16>::value, L::BOX)) return cudaErrorInvalidValue;
    const unsigned blocks = JOIN ? grid.units : (grid.units + L::TEAMS - 1) / L::TEAMS;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(blocks);
    cfg.blockDim = dim3(PR_THREADS);
    cfg.dynamicSmemBytes = L::smem(int(grid.one_keys));
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = unsigned(a.splits);
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = JOIN && grid.cluster ? 1 : 0;
    return cudaLaunchKernelEx(&cfg, paged_rows_kernel<T, HD, RG, NR, JOIN, ONE>, maps, a, grid);
}
template <class T, int HD>
cudaError_t dispatch_rows(const PagedAttention& a, const PagedGrid& grid, const PagedPlan& plan, cudaStream_t stream) {
    if (plan.one) switch (plan.tile_rows) {
        case 8: return launch_rows<T, HD, 1, 1, false, true>(a, grid, stream);
        case 16: return launch_rows<T, HD, 2, 1, false, true>(a, grid, stream);
        case 32: return launch_rows<T, HD, 4, 1, false, true>(a, grid, stream);
        default: return launch_rows<T, HD, 4, 2, false, true>(a, grid, stream);
    }
    const bool join = plan.join;
    switch (plan.tile_rows) {
        case 8: return join ? launch_rows<T, HD, 1, 1, true, false>(a, grid, stream) : launch_rows<T, HD, 1, 1, false, false>(a, grid, stream);
        case 16: return join ? launch_rows<T, HD, 1, 2, true, false>(a, grid, stream) : launch_rows<T, HD, 2, 1, false, false>(a, grid, stream);
        case 32: return join ? launch_rows<T, HD, 2, 2, true, false>(a, grid, stream) : launch_rows<T, HD, 2, 2, false, false>(a, grid, stream);
        default: return launch_rows<T, HD, 4, 2, false, false>(a, grid, stream);     // one team
    }
}

template <class T, int HD, int G>
cudaError_t launch_combine(const PagedAttention& a, const PagedGrid& grid, int tile_rows, cudaStream_t stream) {
    constexpr int ROWS = 128 / (HD / 8 * G);
    const int64_t rows = int64_t(grid.items - grid.whole) * tile_rows;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(unsigned((rows + ROWS - 1) / ROWS));
    cfg.blockDim = dim3(128);
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, paged_combine_kernel<T, HD, G>, a, grid, tile_rows);
}

template <class T, int HD>
cudaError_t dispatch(const PagedAttention& a, const PagedPlan& plan, const PagedGrid& grid, cudaStream_t stream) {
    const cudaError_t e = plan.tiles ? paged_attention_tiles(a, grid, std::is_same<T, __nv_bfloat16>::value, stream)
                                     : dispatch_rows<T, HD>(a, grid, plan, stream);
    if (e != cudaSuccess || a.splits == 1 || grid.cluster) return e;
    return a.splits > 4 ? launch_combine<T, HD, 8>(a, grid, plan.tile_rows, stream) : launch_combine<T, HD, 2>(a, grid, plan.tile_rows, stream);
}

// Blocks of joined teams that the device runs at once in clusters of n: with one block an SM a cluster of
// 8 leaves 28 of the 148 SMs idle, a cluster of 2 none. Asked once for each device and layout.
template <int HD, int RG, int NR>
int cluster_blocks(int n, int dev, int sms) {
    static std::atomic<int> counts[64][8];
    int blocks = counts[dev][n - 1].load(std::memory_order_relaxed);
    if (blocks) return blocks;
    using L = RowsLayout<HD, RG, false>;
    const auto kernel = paged_rows_kernel<__half, HD, RG, NR, true, false>;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(unsigned(n));
    cfg.blockDim = dim3(PR_THREADS);
    cfg.dynamicSmemBytes = L::SMEM;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = unsigned(n);
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    int clusters = 0;
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, L::SMEM) != cudaSuccess ||
        cudaOccupancyMaxActiveClusters(&clusters, kernel, &cfg) != cudaSuccess || clusters < 1) {
        cudaGetLastError();                               // no device: the plan is still one that runs
        return sms * (8 * 64 / HD * RG / 4) * 7 / 8;
    }
    blocks = clusters * n;
    counts[dev][n - 1].store(blocks, std::memory_order_relaxed);
    return blocks;
}

}  // namespace

cudaError_t paged_drain_selftest(int* err, const void* src, cudaStream_t stream) {
    drain_selftest_kernel<<<1, 32, 0, stream>>>(err, static_cast<const uint8_t*>(src));
    return cudaGetLastError();
}

// A tensor map over one of the pools, its axes in order of stride (an axis of one entry has none of
// its own).
static bool page_map(PageMap* at, const void* base, bool bf16, const PagedCache& c, int64_t page, int64_t head, int64_t slot,
                     int box_slots) {
    const int slots = 1 << c.page_shift;
    struct Axis { int64_t stride, size; int box; int* where; } ax[3] = {{slot, slots, std::min(slots, box_slots), &at->slot},
                                                                        {head, c.kv_heads, 1, &at->head},
                                                                        {page, c.num_pages, 1, &at->page}};
    int64_t top = 0;
    for (const Axis& x : ax) top = std::max(top, x.size > 1 ? x.stride * x.size : x.stride);
    for (Axis& x : ax)
        if (x.size == 1) x.stride = top;
    std::stable_sort(ax, ax + 3, [](const Axis& x, const Axis& y) { return x.stride < y.stride; });
    for (int i = 0; i < 3; ++i) *ax[i].where = i + 1;
    return make_map_4d_16bit(&at->map, base, bf16, c.head_dim, {ax[0].size, ax[1].size, ax[2].size},
                             {ax[0].stride, ax[1].stride, ax[2].stride}, {ax[0].box, ax[1].box, ax[2].box});
}
bool page_maps(PageMaps* m, const PagedCache& c, bool bf16, int box_slots) {
    return page_map(&m->k, c.k, bf16, c, c.k_page, c.k_head, c.k_slot, box_slots) &&
           page_map(&m->v, c.v, bf16, c, c.v_page, c.v_head, c.v_slot, box_slots);
}

// Which way to run a call: a figure for each, and the least is taken. It goes by sizes alone (the bounds that the
// host knows; the lengths stand on the device): rounds of units (a problem's keys or a share of them), each with a
// start and its keys, where a unit goes at the rate of its own teams' loads or at its part of what an SM loads,
// whichever is slower. The figures rank the ways and are near microseconds, but are no prediction: the constants
// were fitted to the best choice over even and uneven lengths together, which sets them below what even lengths
// take (kShared of head_dim 128 is twice the memory's rate), and pages count as whole tiles (pages of 64, 16 and
// 8 positions take a decode batch of 64 sequences, 8,192 keys and 8 cached heads of 128 318, 336 and 379 us: a load
// for each page). Fitted to 9,983 calls (1 to 256 rows, 97 to 198,000 keys, 1 to 512 sequences, 2 to 16 cached
// heads, even and uneven lengths), each timed in every way open to it by a build that forces the way: the
// chosen way took 1.02 times the best one's time on average, 1.13 at the 95th percentile, 1.42 at worst; fixed
// bounds on rows and keys (teams joined above 256 keys, tiles above 64 rows) 1.16, 1.75 and 5.6.
// Both sides, us: one row over 500 keys of 64, 24,576 problems: a team each 520, teams joined 604, and
// over 800 keys, 96 problems: 33 and 16; 64 rows over 4,016 keys of 128, 512 problems: rows 303, tiles 242,
// and over 128 keys of 64, 12,288 problems: rows 213, tiles 555; 16 problems over 11,000 keys of 128, clusters
// of 6 and of 8 (one too many for a round): 31 and 45.
struct RowsChoice {
    double us = 0;
    bool join = false;
    int splits = 1;
};
static RowsChoice rows_choice(int tile_rows, int head_dim, int64_t items, int64_t keys, bool one_seq, int64_t sms) {
    const int at = tile_rows == 8 ? 0 : tile_rows == 16 ? 1 : tile_rows == 32 ? 2 : 3;
    const bool wide = head_dim == 128;
    // us a key: of what an SM loads, a problem's part at each size of rows; and of what a team loads
    constexpr double kShared[2][4] = {{.0046, .0046, .0052, .0110}, {.0061, .0074, .0075, .0113}}, kTeam = .0245;
    const double shared = kShared[wide][at];
    const int teams = (wide ? 4 : 8) / (at == 3 ? 2 : 1), joined = at == 3 ? 1 : at == 2 ? 2 : 4;      // of an SM, of a block
    int dev = 0;
    cudaGetDevice(&dev);
    if (dev < 0 || dev >= 64) dev = 0;
    RowsChoice best;
    auto consider = [&](bool join, int64_t splits) {
        const int block = join ? joined : 1;
        const bool cluster = join && splits > 1 && splits <= 8;
        int64_t slots = sms * teams / block;
        if (cluster) {
            const int n = int(splits);
            slots = (wide ? at == 0 ? cluster_blocks<128, 1, 1> : at == 1 ? cluster_blocks<128, 1, 2> : cluster_blocks<128, 2, 2>
                          : at == 0 ? cluster_blocks<64, 1, 1> : at == 1 ? cluster_blocks<64, 1, 2> : cluster_blocks<64, 2, 2>)(n, dev, int(sms));
        }
        const int64_t units = items * splits, rounds = units / slots, rest = units % slots;
        const double start = (join ? 3.7 : 2.9) + (cluster ? 1.1 + .13 * double(splits) : 0);
        auto round = [&](int64_t at_once) {
            return at_once ? start + double(keys) / double(splits) * std::max(kTeam / block, double(at_once) / double(sms) * shared) : 0;
        };
        // uneven lengths and starts leave about a third of a round behind the last, one sequence's starts less (with
        // a third there too 8 problems over 131,072 keys of 128 run as 55 splits each, 92 us; 18 of them: 87)
        double us = double(rounds) * round(slots) + round(rest) + (one_seq ? .2 : .35) * round(rounds ? slots : rest);
        // a second kernel, and the partial rows through the workspace
        if (splits > 1 && !cluster) us += 2.7 + .1 * double(splits) + 4.2e-7 * double(units * tile_rows) * (head_dim * 4 + 8);
        if (best.us == 0 || us < best.us) best = {us, join, int(splits)};
    };
    consider(false, 1);
    const bool join = joined > 1;
    for (int64_t n = join ? 1 : 2; n <= 8 && (n == 1 || keys >= 32 * n); ++n) consider(join, n);
    for (int64_t n = 1; n <= 3; ++n) {
        const int64_t splits = std::min<int64_t>(sms * teams / joined * n / items, 256);
        if (splits > 8 && keys >= 64 * splits) consider(join, splits);
    }
    return best;
}

PagedPlan paged_plan(const PagedAttention& a) {
    PagedPlan p;
    const int64_t rows = int64_t(a.batch.max_chunk) * a.group, problems = int64_t(a.cache.kv_heads) * a.batch.seqs;
    const int64_t sms = device_sm_count();
    const int64_t keys = a.window ? std::min<int64_t>(a.batch.max_length, int64_t(a.window) + a.batch.max_chunk) : a.batch.max_length;
    // Row tiles that hold rows: where the new tokens are uneven, fewer than max_chunk allows (the rest of
    // the grid ends at once). 7 prompts of 1 to 300 tokens, window 1,000, planned as if all of 300: 41 us, so: 37.
    auto held = [&](int64_t row_tiles, int tile_rows) {
        return std::max<int64_t>(std::min(row_tiles * a.batch.seqs, int64_t(a.batch.tokens) * a.group / tile_rows + a.batch.seqs), 1) * a.cache.kv_heads;
    };
    // tiles: as many items as fill the SMs once or more stay whole; the rest are split so that they take
    // the least time together
    int64_t tiles_cost = 0, tiles_whole = 0;
    int tiles_splits = 1;
    if (rows > 8) {                                       // 8 rows are padded to 256: never faster
        const int64_t row_tiles = (rows + kPagedTileRows - 1) / kPagedTileRows, tiles = (keys + 127) / 128;
        const int64_t items = held(row_tiles, kPagedTileRows), rest = items % sms;
        const int64_t all = row_tiles * problems;             // rest of them, or as many more as end at once
        tiles_whole = all - rest * all / items;
        int64_t best = rest ? INT64_MAX : 0;
        for (int s = 1; rest && s <= 32 && (s == 1 || 2 * s <= tiles); ++s) {
            const int64_t cost = (rest * s + sms - 1) / sms * ((tiles + s - 1) / s + 3) + (s > 1 ? 4 : 0);
            if (cost < best) { best = cost; tiles_splits = s; }
        }
        tiles_cost = items / sms * (tiles + 3) + best;
    }
    p.tile_rows = rows_of_team(a);
    p.row_tiles = (rows + p.tile_rows - 1) / p.tile_rows;
    // 96 rows over 96 keys, 6,144 problems: one tile of keys 166 us, tcgen05 285
    p.one = !a.window && a.batch.max_length <= 96 && rows <= kPagedTileRows;
    RowsChoice choice;
    if (!p.one && rows <= kPagedTileRows)
        choice = rows_choice(p.tile_rows, a.cache.head_dim, held(p.row_tiles, p.tile_rows), std::max<int64_t>(keys, 1), a.batch.seqs == 1, sms);
    p.tiles = !p.one && rows > 8 && (rows > kPagedTileRows || choice.us > 4.4 + 1.69 * double(tiles_cost));
    if (p.tiles) {
        p.tile_rows = kPagedTileRows;
        p.row_tiles = (rows + kPagedTileRows - 1) / kPagedTileRows;
        p.whole = tiles_whole;
        p.splits = tiles_splits;
    } else {
        p.join = choice.join;
        p.splits = choice.splits;
        // Up to 8 splits of a problem are a cluster whose blocks join in shared memory; more go through the
        // workspace and a second kernel.
        if (p.join && p.splits > 1) p.cluster = std::min(p.splits, 8);
    }
    p.items = p.row_tiles * problems;
    p.split_bytes = size_t(p.items - p.whole) * p.tile_rows * (size_t(a.cache.head_dim) * 4 + 8);
    return p;
}

void paged_workspace(PagedAttention* a, void* workspace, size_t bytes) {
    const PagedPlan p = paged_plan(*a);
    const size_t held = workspace && p.split_bytes ? bytes / p.split_bytes : 0;
    a->part_o = nullptr;
    a->part_ml = nullptr;
    a->splits = held < 2 ? 1 : int(std::min<size_t>(held, size_t(p.splits)));
    if (p.cluster >= a->splits) a->splits = p.cluster;     // a cluster's blocks join their splits without it
    if (a->splits == 1 || p.cluster == a->splits) return;
    // weighted values, then their (maximum, sum) pairs
    a->part_o = static_cast<float*>(workspace);
    a->part_ml = reinterpret_cast<float2*>(a->part_o + size_t(a->splits) * size_t(p.items - p.whole) * p.tile_rows * a->cache.head_dim);
}

cudaError_t paged_attention(const PagedAttention& a, bool bf16, cudaStream_t stream) {
    const PagedPlan p = paged_plan(a);
    const int64_t whole = a.splits > 1 ? p.whole : p.items, units = whole + (p.items - whole) * a.splits;
    // (asked before the first kernel is on the stream, which the join's grid would be too late for)
    if (units > INT32_MAX - 4 || (a.part_o && (p.items - whole) * p.tile_rows > INT32_MAX - 128)) return cudaErrorInvalidValue;
    PagedGrid g;
    g.splits = FastDiv(uint32_t(a.splits));
    g.heads = FastDiv(uint32_t(a.cache.kv_heads));
    g.seqs = FastDiv(uint32_t(a.batch.seqs));
    g.group = FastDiv(uint32_t(a.group));
    g.items = uint32_t(p.items);
    g.whole = uint32_t(whole);
    g.units = uint32_t(units);
    g.row_tiles = uint32_t(p.row_tiles);
    g.cluster = a.splits > 1 && !a.part_o;
    g.one_keys = uint32_t(std::max(16, (a.batch.max_length + 15) / 16 * 16));
    if (a.cache.head_dim == 64) return bf16 ? dispatch<__nv_bfloat16, 64>(a, p, g, stream) : dispatch<__half, 64>(a, p, g, stream);
    return bf16 ? dispatch<__nv_bfloat16, 128>(a, p, g, stream) : dispatch<__half, 128>(a, p, g, stream);
}

}  // namespace tsb
