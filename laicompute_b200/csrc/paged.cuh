// KV cache in pages: where a position lies, and the append of new rows with
// the position rotation on the way.
//
// A page holds page_size positions of every KV head, [kv_head][position][dim],
// so one (page, head) pair is a contiguous run that attention streams. A
// sequence's page ids stand in its row of the page table. Indices come from
// device memory, so the kernels check each one before they use it: a bad one
// leaves its bit in the cache's error word and the access is skipped.
#pragma once
#include "common.cuh"

namespace laic {

__host__ __device__ inline void kv_flag(int* err, int bits) {
#ifdef __CUDA_ARCH__
    atomicOr(err, bits);
#else
    *err |= bits;
#endif
}

// The page of position `pos` of sequence `seq`, or -1 where an index is out of range (recorded).
// positions: rows of the rotation table (INT_MAX: no rotation).
__host__ __device__ inline int kv_place(int seq, int pos, const int* table, int nseq, int pages_per_seq, int page_shift,
                                        int num_pages, int positions, int& bad) {
    const int at = pos >> page_shift;
    bad = 0;
    if (seq < 0 || seq >= nseq) bad |= kKvBadSeq;
    if (pos < 0 || at >= pages_per_seq || pos >= positions) bad |= kKvBadPos;
    if (bad) return -1;
    const int page = table[(size_t)seq * pages_per_seq + at];
    if (page >= 0 && page < num_pages) return page;
    bad = kKvBadPage;
    return -1;
}

struct KvAppendParams {
    const void *q, *k, *v;
    void* q_out;
    long long ldq, ldk, ldv, ldqo;
    __half *kp, *vp;
    int rows, heads, kv_heads, head_dim, page_shift, num_pages;
    const int *pos, *seq, *table;
    int nseq, pages_per_seq;
    const float2* rope;
    int rope_pairs, rope_positions;
    bool vec_rope;  // rows of the rotation table are 16-byte aligned
    int units;      // eight-element units of a row: (heads + 2 kv_heads) * head_dim / 8
    int* err;
};

template <typename T> __device__ __forceinline__ float kv_in(T x);
template <> __device__ __forceinline__ float kv_in<float>(float x) { return x; }
template <> __device__ __forceinline__ float kv_in<__half>(__half x) { return __half2float(x); }
template <typename T> __device__ __forceinline__ T kv_out(float x);
template <> __device__ __forceinline__ float kv_out<float>(float x) { return x; }
template <> __device__ __forceinline__ __half kv_out<__half>(float x) { return __float2half_rn(x); }

// Eight consecutive elements as loaded; VEC: the address is 16-byte aligned.
template <typename T>
struct Raw8 {
    uint4 w[sizeof(T) / 2];
    __device__ __forceinline__ float at(int i) const { return kv_in<T>(reinterpret_cast<const T*>(w)[i]); }
};
template <typename T, bool VEC>
__device__ __forceinline__ void load8(const T* p, Raw8<T>& r) {
    if constexpr (VEC) {
#pragma unroll
        for (int j = 0; j < (int)sizeof(T) / 2; ++j) r.w[j] = reinterpret_cast<const uint4*>(p)[j];
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) reinterpret_cast<T*>(r.w)[i] = p[i];
    }
}
template <typename T, bool VEC>
__device__ __forceinline__ void store8(T* p, const float (&x)[8]) {
    Raw8<T> r;
#pragma unroll
    for (int i = 0; i < 8; ++i) reinterpret_cast<T*>(r.w)[i] = kv_out<T>(x[i]);
    if constexpr (VEC) {
#pragma unroll
        for (int j = 0; j < (int)sizeof(T) / 2; ++j) reinterpret_cast<uint4*>(p)[j] = r.w[j];
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) p[i] = reinterpret_cast<const T*>(r.w)[i];
    }
}

constexpr int kAppendUnits = 4;  // units per thread and row

// Grid (rows / R, slices of a row). A thread owns whole rotation pairs, so q_out may be q itself; it
// loads all its units of R rows before the chains position -> sequence -> page are resolved, and the
// grid covers many rows per SM: memory bounds long appends (8,188 rows of 32 + 16 heads of 128 in
// binary16: 38 us, 5.3 TB/s, 81 % of a copy's rate), the chain of three loads short ones. The
// rotation is the reference's unfused multiply and add (src/inference_v2.cpp:25) in FP32; k and v are
// rounded to binary16 once, which is the cache's precision.
template <typename TI, typename TQ, bool VEC, int R>
__global__ void __launch_bounds__(256) kv_append_kernel(const KvAppendParams p) {
    const int sh = __ffs(p.head_dim) - 4;  // units per head: 2^sh
    const int u0 = blockIdx.y * blockDim.x * kAppendUnits + threadIdx.x;
    pdl_wait();
    int pos[R], seq[R];
#pragma unroll
    for (int q = 0; q < R; ++q) {
        const int t = blockIdx.x * R + q;
        pos[q] = t < p.rows ? p.pos[t] : -1;
        seq[q] = t < p.rows && p.seq ? p.seq[t] : t;
    }
    Raw8<TI> raw[R][kAppendUnits];
#pragma unroll
    for (int q = 0; q < R; ++q) {
        const int t = blockIdx.x * R + q;
#pragma unroll
        for (int j = 0; j < kAppendUnits; ++j) {
            const int u = u0 + j * blockDim.x;
            if (u < p.units && t < p.rows) {
                const int head = u >> sh, hk = head - p.heads, hv = hk - p.kv_heads;
                const TI* src = hk < 0   ? static_cast<const TI*>(p.q) + (size_t)t * p.ldq + (size_t)u * 8
                                : hv < 0 ? static_cast<const TI*>(p.k) + (size_t)t * p.ldk + (size_t)(u - (p.heads << sh)) * 8
                                         : static_cast<const TI*>(p.v) + (size_t)t * p.ldv +
                                               (size_t)(u - ((p.heads + p.kv_heads) << sh)) * 8;
                load8<TI, VEC>(src, raw[q][j]);
            }
        }
    }
    // the units of a thread lie blockDim.x apart, a whole number of heads: one set of angles per row
    const int d = (u0 & ((1 << sh) - 1)) * 8, pr = d >> 1;
    float2 c[R][4];
    int page[R];
#pragma unroll
    for (int q = 0; q < R; ++q) {
        const float2* cs = p.rope + (size_t)min(max(pos[q], 0), p.rope_positions - 1) * p.rope_pairs;
        if (p.vec_rope && pr + 4 <= p.rope_pairs) {
            *reinterpret_cast<float4*>(c[q]) = __ldg(reinterpret_cast<const float4*>(cs + pr));
            *reinterpret_cast<float4*>(c[q] + 2) = __ldg(reinterpret_cast<const float4*>(cs + pr + 2));
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (pr + i < p.rope_pairs) c[q][i] = __ldg(cs + pr + i);
        }
        int bad = 0;
        page[q] = pos[q] < 0 ? -1 : kv_place(seq[q], pos[q], p.table, p.nseq, p.pages_per_seq, p.page_shift, p.num_pages,
                                             p.rope_positions, bad);
        if (bad && threadIdx.x == 0 && blockIdx.y == 0) kv_flag(p.err, bad);
    }
#pragma unroll
    for (int q = 0; q < R; ++q) {
        if (page[q] < 0) continue;  // padding, or refused
        const int t = blockIdx.x * R + q;
        const int off = pos[q] & ((1 << p.page_shift) - 1);
#pragma unroll
        for (int j = 0; j < kAppendUnits; ++j) {
            const int u = u0 + j * blockDim.x;
            if (u >= p.units) break;
            const int head = u >> sh, hk = head - p.heads, hv = hk - p.kv_heads;
            float x[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] = raw[q][j].at(i);
            if (hv < 0) {
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (pr + i < p.rope_pairs) {
                        const float a = x[2 * i], b = x[2 * i + 1];
                        x[2 * i] = __fsub_rn(__fmul_rn(a, c[q][i].x), __fmul_rn(b, c[q][i].y));
                        x[2 * i + 1] = __fadd_rn(__fmul_rn(a, c[q][i].y), __fmul_rn(b, c[q][i].x));
                    }
            }
            if (hk < 0) {
                store8<TQ, VEC>(static_cast<TQ*>(p.q_out) + (size_t)t * p.ldqo + (size_t)u * 8, x);
            } else {
                const int h = hv < 0 ? hk : hv;
                __half* dst = (hv < 0 ? p.kp : p.vp) +
                              (((((size_t)page[q] * p.kv_heads + h) << p.page_shift) + off) * p.head_dim + d);
                store8<__half, true>(dst, x);  // pages are 16-byte aligned and head_dim a multiple of 8
            }
        }
    }
}

}  // namespace laic
