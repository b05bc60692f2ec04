// Probabilities of logits rows, and the check of drafted tokens against them.
#pragma once
#include <cooperative_groups.h>

#include "common.cuh"
#include "paged_attn.cuh"  // ex2

namespace laic {

// ---------------------------------------------------------------------------
// softmax(logits / T)
// ---------------------------------------------------------------------------
struct ProbsParams {
    const float* x;
    float* y;
    const float* temp;
    long long ldx, ldy;
    int vocab;
};

// 2^((x - m) log2(e) / T) with the product's rounding error carried along: the FP32 difference and
// product alone would lose |exponent| * 2^-24 of the result. k + kl = log2(e) / T.
__device__ __forceinline__ float prob_exp(float x, float m, float k, float kl) {
    const float d = __fsub_rn(x, m);
    const float bb = __fsub_rn(d, x);
    const float e = __fsub_rn(__fsub_rn(x, __fsub_rn(d, bb)), __fadd_rn(m, bb));  // (x - m) - d, exactly
    const float h = __fmul_rn(d, k);
    if (!(h > -150.f)) return 0.f;  // below binary32 (a mask of the lowest value overflows d and h)
    const float l = fmaf(d, kl, fmaf(e, k, fmaf(d, k, -h)));
    const float p = ex2(h);
    return fmaf(p, l * 0.69314718f, p);
}

// One row per CTA, three passes over it (the second and third from L2).
constexpr int kProbsThreads = 1024;
__global__ void __launch_bounds__(kProbsThreads) probs_kernel(const ProbsParams p) {
    __shared__ float red[32];
    __shared__ int redi[32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const float* x = p.x + (size_t)blockIdx.x * p.ldx;
    float* y = p.y + (size_t)blockIdx.x * p.ldy;
    const float t = p.temp[blockIdx.x];
    float m = -INFINITY;
    int at = 0x7fffffff;
    for (int i = threadIdx.x; i < p.vocab; i += kProbsThreads) {
        const float v = x[i];
        if (v > m) { m = v; at = i; }  // NaN never
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        const float om = __shfl_xor_sync(0xffffffffu, m, o);
        const int oa = __shfl_xor_sync(0xffffffffu, at, o);
        if (om > m || (om == m && oa < at)) { m = om; at = oa; }
    }
    if (lane == 0) { red[warp] = m; redi[warp] = at; }
    __syncthreads();
    m = -INFINITY; at = 0x7fffffff;
    for (int w = 0; w < kProbsThreads / 32; ++w)
        if (red[w] > m || (red[w] == m && redi[w] < at)) { m = red[w]; at = redi[w]; }
    __syncthreads();
    if (!(t > 0.f) || m == -INFINITY) {  // greedy: the first maximum; a row of -inf: zeros
        for (int i = threadIdx.x; i < p.vocab; i += kProbsThreads) y[i] = i == at && m != -INFINITY ? 1.f : 0.f;
        return;
    }
    const double kd = 1.4426950408889634 / (double)t;
    const float k = (float)kd, kl = (float)(kd - (double)k);
    auto term = [&](float v) { return m == INFINITY ? (v == INFINITY ? 1.f : 0.f) : v == v && v != -INFINITY ? prob_exp(v, m, k, kl) : 0.f; };
    float s = 0.f;
    for (int i = threadIdx.x; i < p.vocab; i += kProbsThreads) s += term(x[i]);
    s = block_sum(s, red);
    const float iv = 1.f / s;
    for (int i = threadIdx.x; i < p.vocab; i += kProbsThreads) y[i] = term(x[i]) * iv;
}

// ---------------------------------------------------------------------------
// verification of drafted tokens
// ---------------------------------------------------------------------------
struct VerifyParams {
    const float *target, *draft;
    long long ldt, ldd;
    const unsigned* ids;
    const int* n_draft;
    const float *accept_u, *sample_u;
    unsigned* out_ids;
    int* out_n;
    int nseq, max_draft, vocab;
};

constexpr int kVerifyThreads = 512;
constexpr int kVerifyCluster = 8;

__device__ __forceinline__ float prob_in(float x) { return fmaxf(x, 0.f); }  // negative and NaN: 0

// One cluster per sequence. Every CTA finds the first refused token (the numbers are gathered, a
// lane per drafted token), then sums its slice of the row the next token is drawn from; the slices'
// sums meet in distributed shared memory, and the CTA whose slice holds sample_u * total reads it
// once more in order. Sums are in 64 bits: 128k binary32 terms in 32 would move the drawn token.
__global__ void __launch_bounds__(kVerifyThreads) verify_kernel(const VerifyParams p) {
    namespace cg = cooperative_groups;
    cg::cluster_group cluster = cg::this_cluster();
    const int rank = (int)cluster.block_rank(), s = blockIdx.x / kVerifyCluster;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    constexpr int NW = kVerifyThreads / 32;
    __shared__ int s_acc;
    __shared__ double s_sum[2], s_red[NW];
    __shared__ int s_hit, s_last;
    int n = p.n_draft[s];
    if (n < 0) return;  // the whole cluster alike
    n = min(n, p.max_draft);
    const unsigned* ids = p.ids + (size_t)s * p.max_draft;
    if (warp == 0) {
        unsigned no[2];
#pragma unroll
        for (int b = 0; b < 2; ++b) {
            const int j = lane + 32 * b;
            bool refuse = false;
            if (j < n) {
                const unsigned x = ids[j];
                refuse = true;
                if (x < (unsigned)p.vocab) {
                    const float pt = prob_in(p.target[((size_t)s * (p.max_draft + 1) + j) * p.ldt + x]);
                    const float qd = p.draft ? prob_in(p.draft[((size_t)s * p.max_draft + j) * p.ldd + x]) : 1.f;
                    // the product of two binary32 numbers is exact in binary64
                    refuse = !((double)p.accept_u[(size_t)s * p.max_draft + j] * (double)qd < (double)pt);
                }
            }
            no[b] = __ballot_sync(0xffffffffu, refuse);
        }
        if (lane == 0) s_acc = no[0] ? __ffs(no[0]) - 1 : no[1] ? __ffs(no[1]) + 31 : n;
    }
    __syncthreads();
    const int acc = s_acc;
    const float* P = p.target + ((size_t)s * (p.max_draft + 1) + acc) * p.ldt;
    const float* Q = acc < n && p.draft ? p.draft + ((size_t)s * p.max_draft + acc) * p.ldd : nullptr;
    const unsigned hole = acc < n && !p.draft ? ids[acc] : LAIC_NO_TOKEN;  // drafted with certainty: p without it
    int mode = acc < n ? 1 : 0;  // 1: what the draft leaves of p; 0: p itself
    auto value = [&](int v) -> double {
        const float a = prob_in(P[v]);
        if (mode == 0) return (double)a;
        if (Q) return fmax((double)a - (double)prob_in(Q[v]), 0.0);
        return (unsigned)v == hole ? 0.0 : (double)a;
    };
    const int per = ((p.vocab + kVerifyCluster - 1) / kVerifyCluster + 3) & ~3;
    const int v0 = min(p.vocab, rank * per), v1 = min(p.vocab, v0 + per);
    double total = 0.0, before = 0.0;
    int owner = -1;
    for (int pass = 0; pass < 2; ++pass) {
        double a = 0.0;
        for (int v = v0 + tid; v < v1; v += kVerifyThreads) a += value(v);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) a += __shfl_xor_sync(0xffffffffu, a, o);
        if (lane == 0) s_red[warp] = a;
        __syncthreads();
        if (tid == 0) {
            double t = 0.0;
            for (int w = 0; w < NW; ++w) t += s_red[w];
            s_sum[pass] = t;
        }
        cluster.sync();
        double part[kVerifyCluster];
        total = 0.0;
#pragma unroll
        for (int j = 0; j < kVerifyCluster; ++j) {
            part[j] = *cluster.map_shared_rank(&s_sum[pass], j);
            total += part[j];
        }
        if (total > 0.0 || mode == 0) {
            const double t = (double)p.sample_u[s] * total;
            double run = 0.0;
            int last = -1;
            double last_before = 0.0;
#pragma unroll
            for (int j = 0; j < kVerifyCluster; ++j) {
                if (owner < 0 && part[j] > 0.0) {
                    last = j;
                    last_before = run;
                    if (run + part[j] > t) { owner = j; before = run; }
                }
                run += part[j];
            }
            if (owner < 0) { owner = max(last, 0); before = last_before; }  // sample_u at or above one
            break;
        }
        mode = 0;  // the draft leaves nothing: p itself
    }
    cluster.sync();  // every CTA has read the slices' sums
    unsigned* out = p.out_ids + (size_t)s * (p.max_draft + 1);
    if (rank == 0) {
        for (int j = tid; j <= p.max_draft; j += kVerifyThreads)
            if (j != acc) out[j] = j < acc ? ids[j] : LAIC_NO_TOKEN;
        if (tid == 0) p.out_n[s] = acc + 1;
    }
    if (rank != owner) return;
    // the lowest v of this slice whose running sum exceeds t: each thread a run of consecutive
    // elements, the runs' sums scanned, then the run that crosses t walked
    const double t = (double)p.sample_u[s] * total - before;
    const int run_len = (v1 - v0 + kVerifyThreads - 1) / kVerifyThreads;
    const int a0 = min(v1, v0 + tid * run_len), a1 = min(v1, a0 + run_len);
    double mine = 0.0;
    for (int v = a0; v < a1; ++v) mine += value(v);
    double incl = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const double u = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += u;
    }
    if (lane == 31) s_red[warp] = incl;
    if (tid == 0) { s_hit = kVerifyThreads; s_last = -1; }
    __syncthreads();
    double base = 0.0;
    for (int w = 0; w < warp; ++w) base += s_red[w];
    const double end = base + incl;
    if (mine > 0.0) {
        atomicMax(&s_last, tid);
        if (end > t) atomicMin(&s_hit, tid);
    }
    __syncthreads();
    const int who = s_hit < kVerifyThreads ? s_hit : s_last;  // rounding put t at the slice's end: its last element
    if (who < 0) {
        if (tid == 0) out[acc] = 0;  // no positive probability anywhere
        return;
    }
    if (tid != who) return;
    double run = end - mine;
    int pick = a0;
    for (int v = a0; v < a1; ++v) {
        const double x = value(v);
        if (x > 0.0) {
            pick = v;
            run += x;
            if (run > t) break;
        }
    }
    out[acc] = (unsigned)pick;
}

}  // namespace laic
