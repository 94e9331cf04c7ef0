// Operators over a paged cache of keys and values (include/timestral_b200.h): what their
// kernels share. The host entries (paged_api.cu) check the arguments and fill these structs.
#pragma once
#include <cstdint>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include "common.cuh"

namespace tsb {

// Division by a number known at launch: n / d for n < 2^31 as the high word of a product.
struct FastDiv {
    uint32_t d = 1, mul = 0, shift = 0;
    FastDiv() = default;
    explicit FastDiv(uint32_t divisor) : d(divisor) {
        if (d == 1) return;
        while ((1ull << shift) < d) ++shift;                       // mul = ceil(2^(31 + shift) / d) < 2^32
        mul = uint32_t(((1ull << (31 + shift)) + d - 1) / d);
        --shift;
    }
    __device__ __forceinline__ uint32_t div(uint32_t n) const { return d == 1 ? n : __umulhi(n, mul) >> shift; }
    __device__ __forceinline__ uint32_t divmod(uint32_t n, uint32_t* rest) const {
        const uint32_t x = div(n);
        *rest = n - x * d;
        return x;
    }
};

// [tokens][heads][head_dim], strides in elements.
struct PagedHeads {
    void* data = nullptr;
    int64_t token = 0, head = 0;
};

struct PagedRotation {
    const float* cos = nullptr;
    const float* sin = nullptr;
    int64_t stride = 0;
    int rows = 0, dim = 0;
    const int* positions = nullptr;
};

struct PagedCache {
    void* k = nullptr;
    void* v = nullptr;
    int64_t k_page = 0, k_head = 0, k_slot = 0, v_page = 0, v_head = 0, v_slot = 0;
    const int* table = nullptr;
    int64_t table_stride = 0;
    int num_pages = 0, page_shift = 0, kv_heads = 0, head_dim = 0;
};

struct PagedBatch {
    const int* q_start = nullptr;
    const int* lengths = nullptr;
    int seqs = 0, max_chunk = 0, max_length = 0, tokens = 0;
};

struct NormRopeSide {
    PagedHeads in, out;
    const float* weight = nullptr;
    int heads = 0;
    FastDiv units;                      // threads' worth of heads of a token (set by the launch)
};
struct NormRope {
    NormRopeSide q, k;
    PagedRotation rot;
    int tokens = 0, head_dim = 0;
    float eps = 0;
    int* err = nullptr;
};

struct PagedAppend {
    PagedCache cache;
    PagedBatch batch;
    PagedHeads k, v;
    const float* k_weight = nullptr;
    PagedRotation rot;
    float eps = 0;
    int* err = nullptr;
};

struct PagedAttention {
    PagedCache cache;
    PagedBatch batch;
    PagedHeads q, out, gate;
    int q_heads = 0, group = 0, window = 0, self_visible = 0;
    float scale_log2 = 0;               // scale * log2(e)
    const uint32_t* key_valid = nullptr;
    int64_t key_valid_stride = 0;
    int key_valid_positions = 0;
    int splits = 1;                     // of the items behind the grid's first `whole`
    float* part_o = nullptr;            // [items - whole][splits][tile_rows][head_dim], unnormalised
    float2* part_ml = nullptr;          // the same rows: reference maximum (log2 units), sum
    int* err = nullptr;
};

// The work of a call: an item is a tile of rows of one (sequence, cached head), those with the last
// rows (which see most keys) first. The first `whole` items are one unit each, the others a unit for
// each split of their keys.
struct PagedGrid {
    FastDiv splits, heads, seqs, group;
    uint32_t items = 0, whole = 0, units = 0, row_tiles = 0;
    uint32_t one_keys = 0;              // rows, a tile for all keys: the tile's keys
    uint32_t cluster = 0;               // rows: the splits of an item are a cluster
};
struct PagedItem {
    int row_tile, kvh, seq;
};
__device__ __forceinline__ PagedItem item_of(const PagedGrid& g, uint32_t item) {
    uint32_t kvh, seq;
    const uint32_t back = g.seqs.divmod(g.heads.divmod(item, &kvh), &seq);
    return {int(g.row_tiles - 1 - back), int(kvh), int(seq)};
}
// A unit's item, its split, and into how many its item is split.
__device__ __forceinline__ uint32_t unit_of(const PagedGrid& g, uint32_t unit, uint32_t* split, int* splits) {
    if (unit < g.whole) {
        *split = 0;
        *splits = 1;
        return unit;
    }
    *splits = int(g.splits.d);
    return g.whole + g.splits.divmod(unit - g.whole, split);
}

// How a call of paged_attention runs: chosen from sizes alone, so that the workspace query and
// the call agree. splits is what it would like without a bound on the workspace.
struct PagedPlan {
    bool tiles = false;                 // paged_tiles_kernel, else paged_rows_kernel
    bool join = false;                  // rows: a block's teams share one problem
    bool one = false;                   // rows: a tile holds every key
    int tile_rows = 0;
    int64_t row_tiles = 0, items = 0, whole = 0;
    int splits = 1;
    int cluster = 0;                    // splits that need no workspace
    size_t split_bytes = 0;             // workspace bytes of one split
};
PagedPlan paged_plan(const PagedAttention& a);

// Give a call its workspace (or none): as many splits as it holds, its partial results laid out in it.
void paged_workspace(PagedAttention* a, void* workspace, size_t bytes);

// A batch of `seqs` sequences of `length` positions, the last `chunk` of them new, whose pages lie one
// behind the other in the pool, `width` to a sequence.
cudaError_t paged_uniform_batch(int seqs, int chunk, int length, int width, int* q_start, int* lengths, int* table, cudaStream_t stream);
// bf16: values of type bf16, else f16.
cudaError_t norm_rope(const NormRope& a, bool bf16, cudaStream_t stream);
cudaError_t paged_append(const PagedAppend& a, bool bf16, cudaStream_t stream);
cudaError_t paged_attention(const PagedAttention& a, bool bf16, cudaStream_t stream);
// The kernel for many rows (paged_tiles.cu).
cudaError_t paged_attention_tiles(const PagedAttention& a, const PagedGrid& grid, bool bf16, cudaStream_t stream);
constexpr int kPagedTileRows = 256;     // its rows per block

// Test of drain (no fault): err[1] = 1 when it waited for two copies in flight, err[0] = kDevTimeoutAttn when it gave
// up, after one limit, on a phase whose bytes never come all. src: 1 KB of zeros.
cudaError_t paged_drain_selftest(int* err, const void* src, cudaStream_t stream);

// A tensor map over one of the cache's pools: 64 values by up to box_slots slots of one head and
// page, and which coordinate (1, 2 or 3) stands for what, its axes being in order of stride.
struct PageMap {
    CUtensorMap map;
    int slot, head, page;
};
struct PageMaps {
    PageMap k, v;
};
// false when the cache's strides do not fit a tensor map.
bool page_maps(PageMaps* m, const PagedCache& c, bool bf16, int box_slots);

// ---------------------------------------------------------------------------------------
// Device helpers

// 64 values (from x, a multiple of 64) of a box of slots: rows of 128 bytes at dst, 128-byte
// swizzle. A page number outside the pool gives zeros.
__device__ __forceinline__ void load_page(void* dst, const PageMap& m, uint64_t* bar, int x, int slot, int head, int page) {
    const int c1 = m.slot == 1 ? slot : m.head == 1 ? head : page;
    const int c2 = m.slot == 2 ? slot : m.head == 2 ? head : page;
    const int c3 = m.slot == 3 ? slot : m.head == 3 ? head : page;
    tma_load_4d(dst, &m.map, bar, x, c1, c2, c3);
}

// What a block still has in flight when one of its waits ran out lands before the block leaves its shared memory
// (and tensor memory): the `count` phases of a ring of `stages` barriers from (stage, phase) on are complete,
// or, false, one wait limit for all of them is over.
__device__ __forceinline__ bool drain(uint64_t* bars, int stages, int stage, uint32_t phase, int count) {
    const long long start = clock64();
#pragma unroll 1
    for (int i = 0; i < count; ++i) {
        while (!mbar_try_wait(&bars[stage], phase))
            if (clock64() - start > kWaitCycles) return false;
        if (++stage == stages) { stage = 0; phase ^= 1; }
    }
    return true;
}

// The new tokens of sequence s, checked against the bounds the host gave; a contradiction is
// recorded and gives ok = false.
struct SeqInfo { int start, n, len; bool ok; };
__device__ __forceinline__ SeqInfo load_seq(const PagedBatch& b, int s, int* err) {
    SeqInfo q;
    q.start = b.q_start[s];
    const int end = b.q_start[s + 1];
    q.len = b.lengths[s];
    // compared before they are subtracted: any two ints may stand there
    q.ok = q.start >= 0 && end >= q.start && end <= b.tokens && q.len >= 0 && q.len <= b.max_length &&
           end - q.start <= b.max_chunk && end - q.start <= q.len;
    q.n = q.ok ? end - q.start : 0;
    if (!q.ok) record_error(err, kDevBadBatch);
    return q;
}

template <class T>
struct Pair;
template <>
struct Pair<__half> {
    static __device__ __forceinline__ float2 up(uint32_t u) { return __half22float2(*reinterpret_cast<__half2*>(&u)); }
    static __device__ __forceinline__ uint32_t down(float a, float b) {
        const __half2 h = __floats2half2_rn(a, b);
        return *reinterpret_cast<const uint32_t*>(&h);
    }
};
template <>
struct Pair<__nv_bfloat16> {
    static __device__ __forceinline__ float2 up(uint32_t u) {
        return make_float2(__uint_as_float(u << 16), __uint_as_float(u & 0xffff0000u));
    }
    static __device__ __forceinline__ uint32_t down(float a, float b) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
        return *reinterpret_cast<const uint32_t*>(&h);
    }
};
// Probabilities are held as 2^(t - m + lift), m the row's reference maximum, which its largest score passes by
// at most 8: rounded to f16 they reach 2^15 of its 2^16, and what its steps of 2^-24 lose lies 2^-32 below the
// largest. Without the lift 32,768 keys of 2^-26 each behind one that stands out (w = 2^-11 of a row's weight)
// were lost. A power of two changes no other bit, and falls out with the sum. bf16 has the range.
template <class T>
constexpr float kLift = 0.f;
template <>
inline constexpr float kLift<__half> = 7.f;

// Eight 16-bit values <-> floats.
template <class T>
__device__ __forceinline__ void unpack8(const uint4& u, float (&f)[8]) {
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 p = Pair<T>::up(w[i]);
        f[2 * i] = p.x;
        f[2 * i + 1] = p.y;
    }
}
template <class T>
__device__ __forceinline__ uint4 pack8(const float (&f)[8]) {
    return make_uint4(Pair<T>::down(f[0], f[1]), Pair<T>::down(f[2], f[3]), Pair<T>::down(f[4], f[5]),
                      Pair<T>::down(f[6], f[7]));
}

// Keys [k0, k0 + 32) of the sequence whose bits are set (all of them without key_valid).
__device__ __forceinline__ uint32_t valid_word(const PagedAttention& a, int seq, int k0) {
    const int left = a.key_valid_positions - k0;
    if (left <= 0) return ~0u;
    const uint32_t m = a.key_valid[int64_t(seq) * a.key_valid_stride + (k0 >> 5)];
    return left < 32 ? m | ~0u << left : m;
}
// Bits [lo, hi] (inclusive, any ints) of the 32-bit word that starts at bit w0.
__device__ __forceinline__ uint32_t range32(int lo, int hi, int w0) {
    lo = max(lo - w0, 0);
    hi = min(hi - w0, 31);
    if (lo > hi) return 0u;
    return (0xffffffffu >> (31 - hi)) & (0xffffffffu << lo);
}

// Does a new token see one of the positions [from, to), all of which lie where the rows may look? (Asked of
// table entries that name no page: with all of a page's bits clear nobody reads it.)
__device__ __forceinline__ bool any_valid(const PagedAttention& a, int seq, int base, int from, int to) {
    if (!a.key_valid || (a.self_visible && to > base)) return true;
#pragma unroll 1
    for (int k0 = from & ~31; k0 < to; k0 += 32)
        if (valid_word(a, seq, k0) & range32(from, to - 1, k0)) return true;
    return false;
}

}  // namespace tsb
