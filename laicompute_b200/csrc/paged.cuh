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

enum : int { kKvBadSeq = 1, kKvBadPos = 2, kKvBadPage = 4, kKvBadGroup = 8 };

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
    int heads, kv_heads, head_dim, page_shift, num_pages;
    const int *pos, *seq, *table;
    int nseq, pages_per_seq;
    const float2* rope;
    int rope_pairs, rope_positions;
    int* err;
};

template <typename T> __device__ __forceinline__ float kv_in(T x);
template <> __device__ __forceinline__ float kv_in<float>(float x) { return x; }
template <> __device__ __forceinline__ float kv_in<__half>(__half x) { return __half2float(x); }
template <typename T> __device__ __forceinline__ T kv_out(float x);
template <> __device__ __forceinline__ float kv_out<float>(float x) { return x; }
template <> __device__ __forceinline__ __half kv_out<__half>(float x) { return __float2half_rn(x); }

// Eight consecutive elements; VEC: the address is 16-byte aligned.
template <typename T, bool VEC>
__device__ __forceinline__ void load8(const T* p, float (&x)[8]) {
    if constexpr (VEC) {
        constexpr int W = 16 / sizeof(T);
#pragma unroll
        for (int j = 0; j < 8 / W; ++j) {
            const uint4 w = *reinterpret_cast<const uint4*>(p + j * W);
            const T* e = reinterpret_cast<const T*>(&w);
#pragma unroll
            for (int i = 0; i < W; ++i) x[j * W + i] = kv_in<T>(e[i]);
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = kv_in<T>(p[i]);
    }
}
template <typename T, bool VEC>
__device__ __forceinline__ void store8(T* p, const float (&x)[8]) {
    if constexpr (VEC) {
        constexpr int W = 16 / sizeof(T);
#pragma unroll
        for (int j = 0; j < 8 / W; ++j) {
            uint4 w;
            T* e = reinterpret_cast<T*>(&w);
#pragma unroll
            for (int i = 0; i < W; ++i) e[i] = kv_out<T>(x[j * W + i]);
            *reinterpret_cast<uint4*>(p + j * W) = w;
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) p[i] = kv_out<T>(x[i]);
    }
}

// Grid (rows, slices of the row's eight-element units). A thread owns whole
// rotation pairs, so q_out may be q itself. The rotation is the reference's
// unfused multiply and add (src/inference_v2.cpp:25) in FP32; k and v are
// rounded to binary16 once, which is the cache's precision.
template <typename TI, typename TQ, bool VEC>
__global__ void __launch_bounds__(256) kv_append_kernel(const KvAppendParams p) {
    const int t = blockIdx.x;
    const int pos = p.pos[t];
    if (pos < 0) return;
    const int seq = p.seq ? p.seq[t] : t;
    int bad;
    const int page = kv_place(seq, pos, p.table, p.nseq, p.pages_per_seq, p.page_shift, p.num_pages, p.rope_positions, bad);
    if (page < 0) {
        if (threadIdx.x == 0 && blockIdx.y == 0) kv_flag(p.err, bad);
        return;
    }
    const int per_head = p.head_dim >> 3;
    const int units = (p.heads + 2 * p.kv_heads) * per_head;
    const float2* cs = p.rope + (size_t)pos * p.rope_pairs;
    const int off = pos & ((1 << p.page_shift) - 1);
    for (int u = blockIdx.y * blockDim.x + threadIdx.x; u < units; u += blockDim.x * gridDim.y) {
        const int head = u / per_head, d = (u - head * per_head) * 8;
        const bool isq = head < p.heads, isk = !isq && head < p.heads + p.kv_heads;
        const int h = isq ? head : isk ? head - p.heads : head - p.heads - p.kv_heads;
        const TI* src = static_cast<const TI*>(isq ? p.q : isk ? p.k : p.v) + (size_t)t * (isq ? p.ldq : isk ? p.ldk : p.ldv) +
                        (size_t)h * p.head_dim + d;
        float x[8];
        load8<TI, VEC>(src, x);
        if (isq || isk) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int pr = (d >> 1) + i;
                if (pr < p.rope_pairs) {
                    const float2 c = __ldg(cs + pr);
                    const float a = x[2 * i], b = x[2 * i + 1];
                    x[2 * i] = __fsub_rn(__fmul_rn(a, c.x), __fmul_rn(b, c.y));
                    x[2 * i + 1] = __fadd_rn(__fmul_rn(a, c.y), __fmul_rn(b, c.x));
                }
            }
        }
        if (isq) {
            store8<TQ, VEC>(static_cast<TQ*>(p.q_out) + (size_t)t * p.ldqo + (size_t)h * p.head_dim + d, x);
        } else {
            __half* dst = (isk ? p.kp : p.vp) +
                          (((((size_t)page * p.kv_heads + h) << p.page_shift) + off) * p.head_dim + d);
            store8<__half, true>(dst, x);  // pages are 16-byte aligned and head_dim a multiple of 8
        }
    }
}

}  // namespace laic
