// Per-head norm and rotation of queries and keys (norm_rope), and writing keys and values into
// a paged cache with the same norm and rotation on the way (paged_append).
//
// Both read every value once and write it once: the memory rate bounds them. A head is held by
// PT threads (head_dim / 16, rounded up to a power of two), each with two vectors of eight values
// whose elements the rotation pairs (d and d + rope_dim / 2; behind rope_dim two neighbouring
// vectors that nothing turns), so that the rotation needs no exchange and the sum of squares is
// a shuffle over PT lanes.
#include "paged.cuh"

namespace tsb {
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
                                          float eps, int head_dim, bool turned, const float* c, const float* s) {
    if (normed) {
        float ss = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) ss = fmaf(x[i], x[i], fmaf(y[i], y[i], ss));
#pragma unroll
        for (int o = PT / 2; o; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o, PT);
        const float r = 1.0f / sqrtf(ss / float(head_dim) + eps);
#pragma unroll
        for (int i = 0; i < 8; ++i) { x[i] = x[i] * r * w0[i]; y[i] = y[i] * r * w1[i]; }
    }
    if (turned) {
        float cc[8], sn[8];
        *reinterpret_cast<float4*>(cc) = *reinterpret_cast<const float4*>(c);
        *reinterpret_cast<float4*>(cc + 4) = *reinterpret_cast<const float4*>(c + 4);
        *reinterpret_cast<float4*>(sn) = *reinterpret_cast<const float4*>(s);
        *reinterpret_cast<float4*>(sn + 4) = *reinterpret_cast<const float4*>(s + 4);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float a = x[i], b = y[i];
            x[i] = fmaf(a, cc[i], -(b * sn[i]));
            y[i] = fmaf(b, cc[i], a * sn[i]);
        }
    }
}

__device__ __forceinline__ void load_weight(const float* w, int a, int b, float (&w0)[8], float (&w1)[8]) {
#pragma unroll
    for (int i = 0; i < 8; ++i) { w0[i] = w[a + i]; w1[i] = w[b + i]; }
}

constexpr int kThreads = 256;

// blocks [0, q_blocks) norm and turn the queries, the rest the keys. Item = (token, head).
template <class T, int PT, int U>
__global__ void __launch_bounds__(kThreads) norm_rope_kernel(const NormRope a, int q_blocks) {
    const bool is_q = int(blockIdx.x) < q_blocks;
    const NormRopeSide& s = is_q ? a.q : a.k;
    const int64_t block = is_q ? blockIdx.x : int(blockIdx.x) - q_blocks;
    constexpr int HEADS = kThreads / PT;
    const int p = threadIdx.x % PT;
    const int64_t first = block * (HEADS * U) + threadIdx.x / PT, items = int64_t(a.tokens) * s.heads;
    const bool holds = p < a.head_dim / 16;
    int e0, e1;
    pair_at(holds ? p : 0, a.rot.dim, &e0, &e1);
    uint4 u0[U], u1[U];
    int64_t to[U];
    int row[U];
    bool live[U];
#pragma unroll
    for (int j = 0; j < U; ++j) {
        const int64_t item = first + j * HEADS;
        live[j] = item < items && holds;
        row[j] = -1;
        u0[j] = u1[j] = make_uint4(0, 0, 0, 0);
        to[j] = 0;
        if (!live[j]) continue;
        const int64_t token = item / s.heads;
        const int head = int(item - token * s.heads);
        const T* in = static_cast<const T*>(s.in.data) + token * s.in.token + head * s.in.head;
        u0[j] = *reinterpret_cast<const uint4*>(in + e0);
        u1[j] = *reinterpret_cast<const uint4*>(in + e1);
        to[j] = token * s.out.token + head * s.out.head;
        if (a.rot.cos) {
            row[j] = a.rot.positions[token];
            if (row[j] < 0 || row[j] >= a.rot.rows) { record_error(a.err, kDevBadShape); live[j] = false; row[j] = -1; }
        }
    }
    float w0[8] = {}, w1[8] = {};
    if (s.weight && holds) load_weight(s.weight, e0, e1, w0, w1);
#pragma unroll
    for (int j = 0; j < U; ++j) {
        float x[8], y[8];
        unpack8<T>(u0[j], x);
        unpack8<T>(u1[j], y);
        const int64_t at = int64_t(row[j]) * a.rot.stride + e0;
        norm_turn<PT>(x, y, s.weight != nullptr, w0, w1, a.eps, a.head_dim, row[j] >= 0 && e0 < a.rot.dim, a.rot.cos + at,
                      a.rot.sin + at);
        if (!live[j]) continue;
        T* out = static_cast<T*>(s.out.data) + to[j];
        *reinterpret_cast<uint4*>(out + e0) = pack8<T>(x);
        *reinterpret_cast<uint4*>(out + e1) = pack8<T>(y);
    }
}

// One block: the next kThreads / PT (token, head) items of a sequence, its keys and its values.
template <class T, int PT>
__global__ void __launch_bounds__(kThreads) paged_append_kernel(const PagedAppend a, int blocks_per_seq) {
    const int seq = blockIdx.x / blocks_per_seq;
    const SeqInfo q = load_seq(a.batch, seq, a.err);
    const PagedCache& c = a.cache;
    constexpr int HEADS = kThreads / PT;
    const int64_t item = int64_t(blockIdx.x % blocks_per_seq) * HEADS + threadIdx.x / PT;
    const int p = threadIdx.x % PT;
    const int i = int(item / c.kv_heads), head = int(item - int64_t(i) * c.kv_heads);
    const bool live = i < q.n;
    if (!__any_sync(0xffffffffu, live)) return;
    int e0, e1;
    pair_at(p, a.rot.dim, &e0, &e1);
    uint4 k0 = make_uint4(0, 0, 0, 0), k1 = k0, v0 = k0, v1 = k0;
    int page = -1, pos = 0, row = -1;
    bool writes = live;
    if (live) {
        const int64_t token = q.start + i;
        const T* k = static_cast<const T*>(a.k.data) + token * a.k.token + head * a.k.head;
        const T* v = static_cast<const T*>(a.v.data) + token * a.v.token + head * a.v.head;
        pos = q.len - q.n + i;
        page = c.table[int64_t(seq) * c.table_stride + (pos >> c.page_shift)];
        k0 = *reinterpret_cast<const uint4*>(k + e0);
        k1 = *reinterpret_cast<const uint4*>(k + e1);
        v0 = *reinterpret_cast<const uint4*>(v + e0);
        v1 = *reinterpret_cast<const uint4*>(v + e1);
        if (page < 0 || page >= c.num_pages) { record_error(a.err, kDevBadPage); writes = false; }
        if (a.rot.cos) {
            row = a.rot.positions ? a.rot.positions[token] : pos;
            if (row < 0 || row >= a.rot.rows) { record_error(a.err, kDevBadShape); writes = false; row = -1; }
        }
    }
    if (a.k_weight || a.rot.cos) {
        float x[8], y[8], w0[8] = {}, w1[8] = {};
        unpack8<T>(k0, x);
        unpack8<T>(k1, y);
        if (a.k_weight) load_weight(a.k_weight, e0, e1, w0, w1);
        const int64_t at = int64_t(row) * a.rot.stride + e0;
        norm_turn<PT>(x, y, a.k_weight != nullptr, w0, w1, a.eps, c.head_dim, row >= 0 && e0 < a.rot.dim, a.rot.cos + at,
                      a.rot.sin + at);
        k0 = pack8<T>(x);
        k1 = pack8<T>(y);
    }
    if (!writes) return;
    const int slot = pos & ((1 << c.page_shift) - 1);
    T* kd = static_cast<T*>(c.k) + page * c.k_page + head * c.k_head + slot * c.k_slot;
    T* vd = static_cast<T*>(c.v) + page * c.v_page + head * c.v_head + slot * c.v_slot;
    *reinterpret_cast<uint4*>(kd + e0) = k0;
    *reinterpret_cast<uint4*>(kd + e1) = k1;
    *reinterpret_cast<uint4*>(vd + e0) = v0;
    *reinterpret_cast<uint4*>(vd + e1) = v1;
}

template <class T, int PT>
cudaError_t launch_norm_rope(const NormRope& a, cudaStream_t stream) {
    constexpr int U = 2, PER = kThreads / PT * U;
    const int64_t qb = (int64_t(a.tokens) * a.q.heads + PER - 1) / PER, kb = (int64_t(a.tokens) * a.k.heads + PER - 1) / PER;
    if (qb + kb > INT32_MAX) return cudaErrorInvalidValue;
    norm_rope_kernel<T, PT, U><<<unsigned(qb + kb), kThreads, 0, stream>>>(a, int(qb));
    return cudaGetLastError();
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

template <class T, int PT>
cudaError_t launch_append(const PagedAppend& a, cudaStream_t stream) {
    const int64_t per_seq = (int64_t(a.batch.max_chunk) * a.cache.kv_heads + kThreads / PT - 1) / (kThreads / PT);
    if (per_seq * a.batch.seqs > INT32_MAX) return cudaErrorInvalidValue;
    paged_append_kernel<T, PT><<<unsigned(per_seq * a.batch.seqs), kThreads, 0, stream>>>(a, int(per_seq));
    return cudaGetLastError();
}

}  // namespace

cudaError_t norm_rope(const NormRope& a, bool bf16, cudaStream_t stream) {
    return bf16 ? dispatch_norm_rope<__nv_bfloat16>(a, stream) : dispatch_norm_rope<__half>(a, stream);
}

cudaError_t paged_append(const PagedAppend& a, bool bf16, cudaStream_t stream) {
    if (a.cache.head_dim == 64)
        return bf16 ? launch_append<__nv_bfloat16, 4>(a, stream) : launch_append<__half, 4>(a, stream);
    return bf16 ? launch_append<__nv_bfloat16, 8>(a, stream) : launch_append<__half, 8>(a, stream);
}

}  // namespace tsb
