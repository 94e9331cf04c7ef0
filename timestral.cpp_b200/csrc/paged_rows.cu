// Per-head norm and rotation of queries and keys (norm_rope), and writing keys and values into
// a paged cache with the same norm and rotation on the way (paged_append).
//
// Both read every value once and write it once: the memory rate bounds them (other buffers each time: 66 to 68 us and
// 0.78 of the copy rate for norm and rotation of 16,384 tokens of 40 heads of 128; 24.7 us, 0.80, for 64 uneven prompts
// of up to 512 tokens appended; 38.6 us, 0.79, for 32,768 tokens of 12 heads of 64 appended as they are). A head is held by
// PT threads (head_dim / 16, rounded up to a power of two), each with two vectors of eight values
// whose elements the rotation pairs (d and d + rope_dim / 2; behind rope_dim two neighbouring
// vectors that nothing turns), so that the rotation needs no exchange and the sum of squares is
// a shuffle over PT lanes.
#include "paged.cuh"

#include <algorithm>
#include <climits>

namespace tsb {

int device_sm_count();

namespace {

// First element of the two vectors of thread `p` of a head.
__device__ __forceinline__ void pair_at(int p, int rope_dim, int* a, int* b) {
    const int turned = rope_dim >> 4;
    if (p < turned) { *a = 8 * p; *b = 8 * p + (rope_dim >> 1); }
    else { *a = rope_dim + 16 * (p - turned); *b = *a + 8; }
}

// The norm (weight w0, w1 of the two vectors) and the rotation of one head's pair of vectors.
// Every thread of the head's PT lanes takes part (live: it holds values).
template <int PT>
__device__ __forceinline__ void norm_turn(float (&x)[8], float (&y)[8], bool normed, const float (&w0)[8], const float (&w1)[8],
                                          float eps, float inv_dim, bool turned, const float (&cc)[8], const float (&sn)[8]) {
    if (normed) {
        float ss = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) ss = fmaf(x[i], x[i], fmaf(y[i], y[i], ss));
#pragma unroll
        for (int o = PT / 2; o; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o, PT);
        const float r = rsqrtf(fmaf(ss, inv_dim, eps));
#pragma unroll
        for (int i = 0; i < 8; ++i) { x[i] = x[i] * r * w0[i]; y[i] = y[i] * r * w1[i]; }
    }
    if (turned) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float a = x[i], b = y[i];
            x[i] = fmaf(a, cc[i], -(b * sn[i]));
            y[i] = fmaf(b, cc[i], a * sn[i]);
        }
    }
}

__device__ __forceinline__ void load8(const float* p, float (&f)[8]) {
    *reinterpret_cast<float4*>(f) = *reinterpret_cast<const float4*>(p);
    *reinterpret_cast<float4*>(f + 4) = *reinterpret_cast<const float4*>(p + 4);
}

// Sixteen bytes that this call reads (writes) once. HINT: first to leave L2, so that the copies which wait
// there to be written back do not push out what is still to be read. Passes over the same buffers, norm and
// rotation of 16,384 tokens of 40 heads of 128: 61.2 us, without the hint 64.5 (other buffers each time it gains less, 0.4 us); a reader right behind it takes as long
// either way (123.3 and 123.8 with it). 64 prompts of 512 tokens appended with a rotation: 20.6 and 22.9. The
// plain copy goes without (2,048 rows of 16 tokens: 36.4, with it 37.1).
template <bool HINT>
__device__ __forceinline__ uint4 load16(const void* p) {
    if constexpr (HINT) return __ldcs(static_cast<const uint4*>(p));
    else return *static_cast<const uint4*>(p);
}
template <bool HINT>
__device__ __forceinline__ void store16(void* p, const uint4& x) {
    if constexpr (HINT) __stcs(static_cast<uint4*>(p), x);
    else *static_cast<uint4*>(p) = x;
}

constexpr int kThreads = 256;

// Blocks [0, q_blocks) norm and turn the queries, the rest the keys. A thread has U heads of one
// token, which share its angles and weights: their table rows (f32, twice the bytes of a 16-bit head)
// come from L1 once for U heads, and 32 U bytes of values are in flight per thread.
template <class T, int PT, int U>
__global__ void __launch_bounds__(kThreads, 4) norm_rope_kernel(const NormRope a, int q_blocks, float inv_dim) {
    const bool is_q = int(blockIdx.x) < q_blocks;
    const NormRopeSide& s = is_q ? a.q : a.k;
    const uint32_t block = is_q ? blockIdx.x : blockIdx.x - q_blocks;
    const int p = threadIdx.x % PT;
    const uint32_t unit = block * (kThreads / PT) + threadIdx.x / PT;
    uint32_t first;
    const uint32_t token = s.units.divmod(unit, &first);
    first *= U;
    const bool here = token < uint32_t(a.tokens) && p < a.head_dim / 16;
    int e0, e1;
    pair_at(p < a.head_dim / 16 ? p : 0, a.rot.dim, &e0, &e1);
    uint4 u0[U], u1[U];
    const T* in = static_cast<const T*>(s.in.data) + int64_t(token) * s.in.token + first * s.in.head;
#pragma unroll
    for (int j = 0; j < U; ++j) {
        u0[j] = u1[j] = make_uint4(0, 0, 0, 0);
        if (!here || int(first) + j >= s.heads) continue;
        u0[j] = load16<true>(in + j * s.in.head + e0);
        u1[j] = load16<true>(in + j * s.in.head + e1);
    }
    bool writes = here, turned = false;
    float c[8] = {}, sn[8] = {}, w0[8] = {}, w1[8] = {};
    if (here && a.rot.cos) {
        const int row = a.rot.positions[token];
        if (row < 0 || row >= a.rot.rows) { record_error(a.err, kDevBadShape); writes = false; }
        turned = writes && e0 < a.rot.dim;
        if (turned) {
            load8(a.rot.cos + row * a.rot.stride + e0, c);
            load8(a.rot.sin + row * a.rot.stride + e0, sn);
        }
    }
    if (s.weight) {
        load8(s.weight + e0, w0);
        load8(s.weight + e1, w1);
    }
    T* out = static_cast<T*>(s.out.data) + int64_t(token) * s.out.token + first * s.out.head;
#pragma unroll
    for (int j = 0; j < U; ++j) {
        float x[8], y[8];
        unpack8<T>(u0[j], x);
        unpack8<T>(u1[j], y);
        norm_turn<PT>(x, y, s.weight != nullptr, w0, w1, a.eps, inv_dim, turned, c, sn);
        if (!writes || int(first) + j >= s.heads) continue;
        store16<true>(out + j * s.out.head + e0, pack8<T>(x));
        store16<true>(out + j * s.out.head + e1, pack8<T>(y));
    }
}

// A block: new tokens of one sequence, U cached heads a thread, their keys and values.
// PLAIN: neither norm nor rotation, so fewer registers and more blocks an SM.
template <class T, int PT, int U, bool PLAIN>
__global__ void __launch_bounds__(kThreads, PLAIN ? 8 : U == 1 ? 4 : 3)
    paged_append_kernel(const PagedAppend a, const FastDiv blocks, const FastDiv units, float inv_dim) {
    uint32_t in_seq, first;
    const int seq = int(blocks.divmod(blockIdx.x, &in_seq));
    const SeqInfo q = load_seq(a.batch, seq, a.err);
    const PagedCache& c = a.cache;
    const int p = threadIdx.x % PT;
    const int i = int(units.divmod(in_seq * (kThreads / PT) + threadIdx.x / PT, &first));
    first *= U;
    const bool live = i < q.n;
    if (!__any_sync(0xffffffffu, live)) return;
    int e0, e1;
    pair_at(p, a.rot.dim, &e0, &e1);
    const int64_t token = q.start + i;
    const int pos = q.len - q.n + i;
    uint4 k0[U], k1[U], v0[U], v1[U];
    int page = -1;
    if (live) page = c.table[int64_t(seq) * c.table_stride + (pos >> c.page_shift)];
    const T* k = static_cast<const T*>(a.k.data) + token * a.k.token + first * a.k.head;
    const T* v = static_cast<const T*>(a.v.data) + token * a.v.token + first * a.v.head;
#pragma unroll
    for (int j = 0; j < U; ++j) {
        k0[j] = k1[j] = v0[j] = v1[j] = make_uint4(0, 0, 0, 0);
        if (!live || int(first) + j >= c.kv_heads) continue;
        k0[j] = load16<!PLAIN>(k + j * a.k.head + e0);
        k1[j] = load16<!PLAIN>(k + j * a.k.head + e1);
        v0[j] = load16<!PLAIN>(v + j * a.v.head + e0);
        v1[j] = load16<!PLAIN>(v + j * a.v.head + e1);
    }
    bool writes = live;
    if (live && (page < 0 || page >= c.num_pages)) { record_error(a.err, kDevBadPage); writes = false; }
    if constexpr (!PLAIN) {
        float cs[8] = {}, sn[8] = {}, w0[8] = {}, w1[8] = {};
        bool turned = false;
        if (live && a.rot.cos) {
            const int row = a.rot.positions ? a.rot.positions[token] : pos;
            if (row < 0 || row >= a.rot.rows) { record_error(a.err, kDevBadShape); writes = false; }
            turned = writes && e0 < a.rot.dim;
            if (turned) {
                load8(a.rot.cos + row * a.rot.stride + e0, cs);
                load8(a.rot.sin + row * a.rot.stride + e0, sn);
            }
        }
        if (a.k_weight) {
            load8(a.k_weight + e0, w0);
            load8(a.k_weight + e1, w1);
        }
#pragma unroll
        for (int j = 0; j < U; ++j) {
            float x[8], y[8];
            unpack8<T>(k0[j], x);
            unpack8<T>(k1[j], y);
            norm_turn<PT>(x, y, a.k_weight != nullptr, w0, w1, a.eps, inv_dim, turned, cs, sn);
            k0[j] = pack8<T>(x);
            k1[j] = pack8<T>(y);
        }
    }
    if (!writes) return;
    const int slot = pos & ((1 << c.page_shift) - 1);
    T* kd = static_cast<T*>(c.k) + page * c.k_page + first * c.k_head + slot * c.k_slot;
    T* vd = static_cast<T*>(c.v) + page * c.v_page + first * c.v_head + slot * c.v_slot;
#pragma unroll
    for (int j = 0; j < U; ++j) {
        if (int(first) + j >= c.kv_heads) break;
        store16<!PLAIN>(kd + j * c.k_head + e0, k0[j]);
        store16<!PLAIN>(kd + j * c.k_head + e1, k1[j]);
        store16<!PLAIN>(vd + j * c.v_head + e0, v0[j]);
        store16<!PLAIN>(vd + j * c.v_head + e1, v1[j]);
    }
}

__global__ void uniform_batch_kernel(int seqs, int chunk, int length, int width, int* q_start, int* lengths, int* table) {
    const int64_t i = int64_t(blockIdx.x) * blockDim.x + threadIdx.x;
    if (i <= seqs) q_start[i] = int(i) * chunk;
    if (i < seqs) lengths[i] = length;
    if (i < int64_t(seqs) * width) table[i] = int(i);
}

template <class T, int PT, int U>
cudaError_t launch_norm_rope(const NormRope& a, cudaStream_t stream) {
    constexpr int PER = kThreads / PT;
    NormRope n = a;
    int64_t blocks[2];
    NormRopeSide* side[2] = {&n.q, &n.k};
    for (int i = 0; i < 2; ++i) {
        const int64_t units = (side[i]->heads + U - 1) / U;
        side[i]->units = FastDiv(uint32_t(units > 0 ? units : 1));
        blocks[i] = (units * a.tokens + PER - 1) / PER;
    }
    if ((blocks[0] + blocks[1]) * PER > INT32_MAX) return cudaErrorInvalidValue;
    norm_rope_kernel<T, PT, U><<<unsigned(blocks[0] + blocks[1]), kThreads, 0, stream>>>(n, int(blocks[0]), 1.0f / float(a.head_dim));
    return cudaGetLastError();
}
template <class T, int PT>
cudaError_t launch_norm_rope(const NormRope& a, cudaStream_t stream) {
    // few tokens: a thread a head, for the latency; else two heads a thread where there are as many (32,768 tokens
    // of 24 heads of 64: 37.4 us, four heads and three blocks an SM 39.4, one head 45.1)
    const int64_t heads = int64_t(a.tokens) * (a.q.heads + a.k.heads);
    return std::max(a.q.heads, a.k.heads) >= 2 && heads * PT >= device_sm_count() * int64_t(2048) ? launch_norm_rope<T, PT, 2>(a, stream)
                                                                           : launch_norm_rope<T, PT, 1>(a, stream);
}
template <class T>
cudaError_t dispatch_norm_rope(const NormRope& a, cudaStream_t stream) {
    const int n = a.head_dim / 16;
    if (n <= 1) return launch_norm_rope<T, 1>(a, stream);
    if (n <= 2) return launch_norm_rope<T, 2>(a, stream);
    if (n <= 4) return launch_norm_rope<T, 4>(a, stream);
    if (n <= 8) return launch_norm_rope<T, 8>(a, stream);
    return launch_norm_rope<T, 16>(a, stream);
}

template <class T, int PT, int U, bool PLAIN>
cudaError_t launch_append(const PagedAppend& a, cudaStream_t stream) {
    const int64_t units = (a.cache.kv_heads + U - 1) / U;
    const int64_t per_seq = (int64_t(a.batch.max_chunk) * units + kThreads / PT - 1) / (kThreads / PT);
    if (per_seq * a.batch.seqs > INT32_MAX || per_seq * (kThreads / PT) > INT32_MAX) return cudaErrorInvalidValue;
    paged_append_kernel<T, PT, U, PLAIN><<<unsigned(per_seq * a.batch.seqs), kThreads, 0, stream>>>(a, FastDiv(uint32_t(per_seq)), FastDiv(uint32_t(units)),
                                                                                               1.0f / float(a.cache.head_dim));
    return cudaGetLastError();
}
template <class T, int PT>
cudaError_t launch_append(const PagedAppend& a, cudaStream_t stream) {
    // a plain copy: a head a thread and all the blocks an SM holds (2,048 rows of 16 tokens: 1.3 us less than with two
    // heads a thread and five blocks an SM); else two heads where there is work for all SMs
    if (!a.k_weight && !a.rot.cos) return launch_append<T, PT, 1, true>(a, stream);
    const bool two = a.cache.kv_heads >= 2 && int64_t(a.batch.max_chunk) * a.batch.seqs * a.cache.kv_heads * PT >= device_sm_count() * int64_t(2048);
    return two ? launch_append<T, PT, 2, false>(a, stream) : launch_append<T, PT, 1, false>(a, stream);
}

}  // namespace

cudaError_t paged_uniform_batch(int seqs, int chunk, int length, int width, int* q_start, int* lengths, int* table, cudaStream_t stream) {
    const int64_t n = std::max(int64_t(seqs) + 1, int64_t(seqs) * width);
    if (n > INT32_MAX || int64_t(seqs) * chunk > INT32_MAX) return cudaErrorInvalidValue;
    uniform_batch_kernel<<<unsigned((n + kThreads - 1) / kThreads), kThreads, 0, stream>>>(seqs, chunk, length, width, q_start, lengths, table);
    return cudaGetLastError();
}

cudaError_t norm_rope(const NormRope& a, bool bf16, cudaStream_t stream) {
    return bf16 ? dispatch_norm_rope<__nv_bfloat16>(a, stream) : dispatch_norm_rope<__half>(a, stream);
}

cudaError_t paged_append(const PagedAppend& a, bool bf16, cudaStream_t stream) {
    if (a.cache.head_dim == 64)
        return bf16 ? launch_append<__nv_bfloat16, 4>(a, stream) : launch_append<__half, 4>(a, stream);
    return bf16 ? launch_append<__nv_bfloat16, 8>(a, stream) : launch_append<__half, 8>(a, stream);
}

}  // namespace tsb
