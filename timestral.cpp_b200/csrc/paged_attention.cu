// Attention of new tokens over a paged cache (tsb_paged_attention): causal, grouped heads, sliding
// window, key-valid bits, optional gate.
//
// out = gate * sum_j p_j v_j / sum_j p_j with p_j = 2^(t_j - m), t_j = (q . k_j) * scale * log2(e),
// m a running maximum: one pass over the keys that keeps m, the sum and the weighted values in f32.
// The rows of one (sequence, cached head) problem are its (token, query head of the group) pairs,
// row = token * group + head, so that a cached key is read once for the whole group.
#include "paged.cuh"

#include <algorithm>
#include <climits>

namespace tsb {

int device_sm_count();

namespace {

// ---------------------------------------------------------------------------------------
// Few rows (single tokens, short chunks): 16 * RG rows a block on mma.sync, bound by the bytes of
// the cache. Four warps: RG row groups of 16 rows, 4 / RG key groups that share each 64-key tile
// out; tiles come in a ring by 16-byte cp.async, in which a key that no row sees (behind the
// length, outside the window, its bit clear) is filled with zeros and not read, so that neither
// its bytes nor what stands there matter. tcgen05 would pad 16 rows to 128 and has nothing to win.
constexpr int PR_THREADS = 128;
constexpr int PR_KT = 64;

template <int HD>
struct RowsLayout {
    static constexpr int STAGES = HD == 64 ? 4 : 3;
    static constexpr int TILE = PR_KT * HD * 2;             // bytes of one tile of keys (or values)
    static constexpr int SMEM = STAGES * 2 * TILE;
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
__device__ __forceinline__ void ldsm4_t(uint32_t addr, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
// 16 bytes, or zeros without reading `src`.
__device__ __forceinline__ void cp_async16_if(uint32_t dst, const void* src, bool read) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(read ? 16 : 0) : "memory");
}

// What one block of rows works on.
struct RowTile {
    int seq, kvh, m0, rows;      // first row and live rows of the tile
    int base;                    // position of the sequence's first new token
    int lo, hi;                  // keys that any row of the tile may see
    int len;                     // length of the sequence
    int start;                   // first token row
};

template <class T, int HD>
__device__ __forceinline__ void load_tile(const PagedAttention& a, const RowTile& t, int k0, uint32_t sk, uint32_t sv) {
    constexpr int CH = HD / 8, STEP = PR_THREADS / CH;
    const PagedCache& c = a.cache;
    const int chunk = threadIdx.x % CH;
    const uint64_t valid = valid_bits(a, t.seq, k0);
    const int slots = 1 << c.page_shift;
    const int* table = c.table + int64_t(t.seq) * c.table_stride;
#pragma unroll
    for (int i = 0; i < PR_KT / STEP; ++i) {
        const int r = threadIdx.x / CH + i * STEP, key = k0 + r;
        bool read = key >= t.lo && key < t.hi && (((valid >> r) & 1) || (a.self_visible && key >= t.base));
        int page = 0;
        if (read) {
            page = table[key >> c.page_shift];
            if (page < 0 || page >= c.num_pages) { record_error(a.err, kDevBadPage); read = false; page = 0; }
        }
        const int slot = key & (slots - 1);
        const T* k = static_cast<const T*>(c.k) + page * c.k_page + t.kvh * c.k_head + slot * c.k_slot + chunk * 8;
        const T* v = static_cast<const T*>(c.v) + page * c.v_page + t.kvh * c.v_head + slot * c.v_slot + chunk * 8;
        const uint32_t at = uint32_t(r * HD * 2 + ((chunk ^ (r & 7)) << 4));
        cp_async16_if(sk + at, k, read);
        cp_async16_if(sv + at, v, read);
    }
}

// Whether the token at position pos sees key.
__device__ __forceinline__ bool sees(const PagedAttention& a, int key, int pos, bool valid) {
    return key <= pos && (a.window == 0 || key > pos - a.window) && (valid || (a.self_visible && key == pos));
}

template <class T, int HD, int RG>
__global__ void __launch_bounds__(PR_THREADS) paged_rows_kernel(const PagedAttention a, int row_tiles) {
    extern __shared__ __align__(1024) uint8_t smem[];
    using L = RowsLayout<HD>;
    constexpr int KG = 4 / RG, KW = PR_KT / KG, NT = KW / 8, KS = HD / 16, ON = HD / 8, MT = 16 * RG;
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, rg = warp % RG, kg = warp / RG;

    RowTile t;
    const int split = int(blockIdx.x % a.splits);
    {
        int b = int(blockIdx.x / a.splits);
        t.m0 = (b % row_tiles) * MT;
        b /= row_tiles;
        t.kvh = b % a.cache.kv_heads;
        t.seq = b / a.cache.kv_heads;
    }
    const SeqInfo q = load_seq(a.batch, t.seq, a.err);
    t.rows = min(MT, q.n * a.group - t.m0);
    if (t.rows <= 0) return;
    t.start = q.start;
    t.len = q.len;
    t.base = q.len - q.n;
    const int t_first = t.m0 / a.group, t_last = (t.m0 + t.rows - 1) / a.group;
    t.hi = t.base + t_last + 1;
    t.lo = a.window ? max(0, t.base + t_first - a.window + 1) : 0;
    // this block's share of the 64-key tiles
    const int tile0 = t.lo / PR_KT, tiles = (t.hi + PR_KT - 1) / PR_KT - tile0;
    const int share = (tiles + a.splits - 1) / a.splits;
    const int first = tile0 + split * share, last = min(first + share, tile0 + tiles);

    // The two rows of this thread, and their tokens' positions (rows that are not there: a
    // position before every key).
    int pos[2];
    int64_t row_at[2];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        const int r = rg * 16 + lane / 4 + 8 * j;
        const int m = t.m0 + r, tok = m / a.group;
        pos[j] = r < t.rows ? t.base + tok : -1;
        row_at[j] = r < t.rows ? (t.start + tok) * a.q.token + (t.kvh * a.group + m - tok * a.group) * a.q.head : -1;
    }
    uint32_t qf[KS][4];
#pragma unroll
    for (int k = 0; k < KS; ++k)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const T* p = static_cast<const T*>(a.q.data) + row_at[j & 1] + k * 16 + (j >> 1) * 8 + (lane & 3) * 2;
            qf[k][j] = row_at[j & 1] >= 0 ? *reinterpret_cast<const uint32_t*>(p) : 0u;
        }

    float o[ON][4];
#pragma unroll
    for (int n = 0; n < ON; ++n) o[n][0] = o[n][1] = o[n][2] = o[n][3] = 0.f;
    float mx[2] = {-INFINITY, -INFINITY}, sum[2] = {0.f, 0.f};

    const uint32_t sbase = smem_u32(smem);
    for (int s = 0; s < L::STAGES - 1; ++s) {
        if (first + s < last) load_tile<T, HD>(a, t, (first + s) * PR_KT, sbase + s * 2 * L::TILE, sbase + s * 2 * L::TILE + L::TILE);
        cp_async_commit();
    }
    int st = 0;
    for (int tile = first; tile < last; ++tile) {
        cp_async_wait<L::STAGES - 2>();
        __syncthreads();
        {   // the stage read last may be loaded again
            const int nx = tile + L::STAGES - 1, ns = (st + L::STAGES - 1) % L::STAGES;
            if (nx < last) load_tile<T, HD>(a, t, nx * PR_KT, sbase + ns * 2 * L::TILE, sbase + ns * 2 * L::TILE + L::TILE);
            cp_async_commit();
        }
        const uint32_t sk = sbase + st * 2 * L::TILE, sv = sk + L::TILE;
        st = (st + 1) % L::STAGES;
        const int k0 = tile * PR_KT + kg * KW;
        float sc[NT][4];
#pragma unroll
        for (int n = 0; n < NT; ++n) sc[n][0] = sc[n][1] = sc[n][2] = sc[n][3] = 0.f;
#pragma unroll
        for (int k = 0; k < KS; ++k)
#pragma unroll
            for (int n = 0; n < NT; n += 2) {
                const int r = kg * KW + n * 8 + (lane & 7) + ((lane >> 4) << 3), ch = 2 * k + ((lane >> 3) & 1);
                uint32_t b[4];
                ldsm4(sk + r * HD * 2 + ((ch ^ (r & 7)) << 4), b);
                mma16816<T>(sc[n], qf[k], b[0], b[1]);
                mma16816<T>(sc[n + 1], qf[k], b[2], b[3]);
            }
        // every row of the tile sees every key of it: no per-key masks
        const uint64_t valid = valid_bits(a, t.seq, tile * PR_KT);
        const bool all = tile * PR_KT + PR_KT - 1 <= t.base + t_first && valid == ~0ull &&
                         (a.window == 0 || tile * PR_KT > t.base + t_last - a.window);
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                sc[n][e] *= a.scale_log2;
                if (!all) {
                    const int key = k0 + n * 8 + (lane & 3) * 2 + (e & 1);
                    if (!sees(a, key, pos[e >> 1], (valid >> (key & 63)) & 1)) sc[n][e] = -INFINITY;
                }
            }
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            float m = mx[j];
#pragma unroll
            for (int n = 0; n < NT; ++n) m = fmaxf(m, fmaxf(sc[n][2 * j], sc[n][2 * j + 1]));
            m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 1));
            m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 2));
            const float ref = m == -INFINITY ? 0.f : m, f = exp2_ftz(mx[j] - ref);
            mx[j] = m;
            float ps = 0.f;
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                sc[n][2 * j] = exp2_ftz(sc[n][2 * j] - ref);
                sc[n][2 * j + 1] = exp2_ftz(sc[n][2 * j + 1] - ref);
                ps += sc[n][2 * j] + sc[n][2 * j + 1];
            }
            sum[j] = fmaf(sum[j], f, ps);
#pragma unroll
            for (int n = 0; n < ON; ++n) { o[n][2 * j] *= f; o[n][2 * j + 1] *= f; }
        }
#pragma unroll
        for (int n = 0; n < NT; n += 2) {
            const uint32_t p[4] = {Pair<T>::down(sc[n][0], sc[n][1]), Pair<T>::down(sc[n][2], sc[n][3]),
                                   Pair<T>::down(sc[n + 1][0], sc[n + 1][1]), Pair<T>::down(sc[n + 1][2], sc[n + 1][3])};
#pragma unroll
            for (int d = 0; d < ON; d += 2) {
                const int r = kg * KW + n * 8 + (lane & 15), ch = d + (lane >> 4);
                uint32_t b[4];
                ldsm4_t(sv + r * HD * 2 + ((ch ^ (r & 7)) << 4), b);
                mma16816<T>(o[d], p, b[0], b[1]);
                mma16816<T>(o[d + 1], p, b[2], b[3]);
            }
        }
    }
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        sum[j] += __shfl_xor_sync(0xffffffffu, sum[j], 1);
        sum[j] += __shfl_xor_sync(0xffffffffu, sum[j], 2);
    }
    // Join the key groups through shared memory: per warp 16 rows of HD f32 (four columns of
    // every row turned by the row, against bank conflicts), maximum and sum.
    cp_async_wait_all();
    __syncthreads();
    float* so = reinterpret_cast<float*>(smem) + warp * 16 * HD;
    float2* sml = reinterpret_cast<float2*>(smem + 4 * 16 * HD * 4);
#pragma unroll
    for (int n = 0; n < ON; ++n)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const int r = lane / 4 + 8 * j, col = n * 8 + (lane & 3) * 2;
            *reinterpret_cast<float2*>(so + r * HD + (col ^ ((r & 7) << 3))) = make_float2(o[n][2 * j], o[n][2 * j + 1]);
        }
    if ((lane & 3) == 0)
#pragma unroll
        for (int j = 0; j < 2; ++j) sml[warp * 16 + lane / 4 + 8 * j] = make_float2(mx[j], sum[j]);
    __syncthreads();
    constexpr int CH = HD / 8;
    for (int i = threadIdx.x; i < t.rows * CH; i += PR_THREADS) {
        const int r = i / CH, c = i % CH, g = r / 16, rr = r % 16;
        float m = -INFINITY;
#pragma unroll
        for (int k = 0; k < KG; ++k) m = fmaxf(m, sml[(k * RG + g) * 16 + rr].x);
        float y[8] = {}, l = 0.f;
#pragma unroll
        for (int k = 0; k < KG; ++k) {
            const int w = k * RG + g;
            const float2 ml = sml[w * 16 + rr];
            const float f = ml.x == -INFINITY ? 0.f : exp2_ftz(ml.x - m);
            l = fmaf(ml.y, f, l);
            const float* src = reinterpret_cast<const float*>(smem) + w * 16 * HD + rr * HD + ((c ^ (rr & 7)) << 3);
#pragma unroll
            for (int e = 0; e < 8; ++e) y[e] = fmaf(src[e], f, y[e]);
        }
        const int row = t.m0 + r, tok = row / a.group, head = t.kvh * a.group + row - tok * a.group;
        const int64_t token = t.start + tok;
        if (a.splits > 1) {
            const int64_t at = int64_t(split) * a.batch.tokens * a.q_heads + token * a.q_heads + head;
            if (c == 0) a.part_ml[at] = make_float2(m, l);
            if (m != -INFINITY) {
                float4* dst = reinterpret_cast<float4*>(a.part_o + at * HD + c * 8);
                dst[0] = make_float4(y[0], y[1], y[2], y[3]);
                dst[1] = make_float4(y[4], y[5], y[6], y[7]);
            }
            continue;
        }
        const float inv = m == -INFINITY ? 0.f : 1.0f / l;
#pragma unroll
        for (int e = 0; e < 8; ++e) y[e] *= inv;
        if (a.gate.data) {
            float gt[8];
            unpack8<T>(*reinterpret_cast<const uint4*>(static_cast<const T*>(a.gate.data) + token * a.gate.token + head * a.gate.head + c * 8), gt);
#pragma unroll
            for (int e = 0; e < 8; ++e) y[e] *= gt[e];
        }
        *reinterpret_cast<uint4*>(static_cast<T*>(a.out.data) + token * a.out.token + head * a.out.head + c * 8) = pack8<T>(y);
    }
}

// Join the splits: item = (new token, query head) of a sequence, HD / 8 threads each.
template <class T, int HD>
__global__ void __launch_bounds__(128) paged_combine_kernel(const PagedAttention a, int blocks_per_seq) {
    constexpr int CH = HD / 8, PER = 128 / CH;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int seq = blockIdx.x / blocks_per_seq;
    const SeqInfo q = load_seq(a.batch, seq, nullptr);
    const int64_t item = int64_t(blockIdx.x % blocks_per_seq) * PER + threadIdx.x / CH;
    const int c = threadIdx.x % CH;
    const int i = int(item / a.q_heads), head = int(item - int64_t(i) * a.q_heads);
    if (i >= q.n) return;
    const int64_t token = q.start + i, at = token * a.q_heads + head, step = int64_t(a.batch.tokens) * a.q_heads;
    float m = -INFINITY;
    for (int s = 0; s < a.splits; ++s) m = fmaxf(m, a.part_ml[s * step + at].x);
    float y[8] = {}, l = 0.f;
    for (int s = 0; s < a.splits; ++s) {
        const float2 ml = a.part_ml[s * step + at];
        if (ml.x == -INFINITY) continue;              // saw nothing: no partial row was written
        const float f = exp2_ftz(ml.x - m);
        l = fmaf(ml.y, f, l);
        const float4* src = reinterpret_cast<const float4*>(a.part_o + (s * step + at) * HD + c * 8);
        const float4 u = src[0], w = src[1];
        y[0] = fmaf(u.x, f, y[0]); y[1] = fmaf(u.y, f, y[1]); y[2] = fmaf(u.z, f, y[2]); y[3] = fmaf(u.w, f, y[3]);
        y[4] = fmaf(w.x, f, y[4]); y[5] = fmaf(w.y, f, y[5]); y[6] = fmaf(w.z, f, y[6]); y[7] = fmaf(w.w, f, y[7]);
    }
    const float inv = m == -INFINITY ? 0.f : 1.0f / l;
#pragma unroll
    for (int e = 0; e < 8; ++e) y[e] *= inv;
    if (a.gate.data) {
        float gt[8];
        unpack8<T>(*reinterpret_cast<const uint4*>(static_cast<const T*>(a.gate.data) + token * a.gate.token + head * a.gate.head + c * 8), gt);
#pragma unroll
        for (int e = 0; e < 8; ++e) y[e] *= gt[e];
    }
    *reinterpret_cast<uint4*>(static_cast<T*>(a.out.data) + token * a.out.token + head * a.out.head + c * 8) = pack8<T>(y);
}

int rows_group(const PagedAttention& a) {
    const int64_t rows = int64_t(a.batch.max_chunk) * a.group;
    return rows <= 16 ? 1 : rows <= 32 ? 2 : 4;
}

template <class T, int HD, int RG>
cudaError_t launch_rows(const PagedAttention& a, cudaStream_t stream) {
    using L = RowsLayout<HD>;
    static KernelSetup configured;
    int dev = 0;
    cudaGetDevice(&dev);
    unsigned long long key = 0;
    if (configured.needed(dev, &key)) {
        const cudaError_t e = cudaFuncSetAttribute(paged_rows_kernel<T, HD, RG>, cudaFuncAttributeMaxDynamicSharedMemorySize, L::SMEM);
        if (e != cudaSuccess) return e;
        configured.done(dev, key);
    }
    const int64_t row_tiles = (int64_t(a.batch.max_chunk) * a.group + 16 * RG - 1) / (16 * RG);
    const int64_t blocks = row_tiles * a.cache.kv_heads * a.batch.seqs;
    if (blocks * a.splits > INT32_MAX) return cudaErrorInvalidValue;
    paged_rows_kernel<T, HD, RG><<<unsigned(blocks * a.splits), PR_THREADS, L::SMEM, stream>>>(a, int(row_tiles));
    return cudaGetLastError();
}

template <class T, int HD>
cudaError_t launch_combine(const PagedAttention& a, cudaStream_t stream) {
    constexpr int PER = 128 / (HD / 8);
    const int64_t per_seq = (int64_t(a.batch.max_chunk) * a.q_heads + PER - 1) / PER;
    if (per_seq * a.batch.seqs > INT32_MAX) return cudaErrorInvalidValue;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(unsigned(per_seq * a.batch.seqs));
    cfg.blockDim = dim3(128);
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, paged_combine_kernel<T, HD>, a, int(per_seq));
}

template <class T, int HD>
cudaError_t dispatch(const PagedAttention& a, cudaStream_t stream) {
    bool taken = false;
    cudaError_t e = cudaSuccess;
    if (paged_plan(a).tiles) e = paged_attention_tiles(a, std::is_same<T, __nv_bfloat16>::value, stream, &taken);
    if (!taken) {
        const int rg = rows_group(a);
        e = rg == 1 ? launch_rows<T, HD, 1>(a, stream) : rg == 2 ? launch_rows<T, HD, 2>(a, stream) : launch_rows<T, HD, 4>(a, stream);
    }
    if (e != cudaSuccess || a.splits == 1) return e;
    return launch_combine<T, HD>(a, stream);
}

}  // namespace

PagedPlan paged_plan(const PagedAttention& a) {
    PagedPlan p;
    p.tiles = int64_t(a.batch.max_chunk) * a.group > 64;
    const int mt = p.tiles ? kPagedTileRows : 16 * rows_group(a), tile = p.tiles ? 128 : 64;
    const int64_t blocks = (int64_t(a.batch.max_chunk) * a.group + mt - 1) / mt * a.cache.kv_heads * a.batch.seqs;
    const int keys = a.window ? int(std::min<int64_t>(a.batch.max_length, int64_t(a.window) + a.batch.max_chunk)) : a.batch.max_length;
    const int64_t want = int64_t(device_sm_count()) * (p.tiles ? 1 : 2);
    p.splits = int(std::max<int64_t>(1, std::min<int64_t>({(want + blocks - 1) / blocks, (keys + 4 * tile - 1) / (4 * tile), 256})));
    p.split_bytes = size_t(a.batch.tokens) * a.q_heads * (size_t(a.cache.head_dim) * 4 + 8);
    return p;
}

cudaError_t paged_attention(const PagedAttention& a, bool bf16, cudaStream_t stream) {
    if (a.cache.head_dim == 64) return bf16 ? dispatch<__nv_bfloat16, 64>(a, stream) : dispatch<__half, 64>(a, stream);
    return bf16 ? dispatch<__nv_bfloat16, 128>(a, stream) : dispatch<__half, 128>(a, stream);
}

}  // namespace tsb
