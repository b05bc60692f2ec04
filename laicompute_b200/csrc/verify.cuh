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

// log2(e) / T as hi + lo: the lo part matters, an error of the factor tilts the whole row. An infinite T
// makes all finite logits alike; one below the smallest normal number counts as that.
struct ProbFactor {
    float k = 0.f, kl = 0.f;
    __device__ __forceinline__ explicit ProbFactor(float t) {
        if (t == INFINITY) return;
        t = fmaxf(t, 0x1p-126f);
        k = 1.44269502f / t;  // log2(e) = 1.44269502162933 (binary32) + 1.9259630e-8
        kl = (fmaf(-k, t, 1.44269502f) + 1.9259630e-8f) / t;
    }
};
// The weight of logit x against the slice's maximum m, 2^(x k - c0): c0 is m k to a 1024th, so that c0 + n
// is exact for the nearest integer n of the exponent and the fraction f = x k - (c0 + n) is rounded at
// its own size (2^-26), not at the exponent's. `off` takes 2^(m k - c0), the same for the whole slice,
// out again. A NaN counts as -inf. Maxima too large for that take the difference first.
struct ProbExp {
    float k, kl, c0, m, off;
    bool huge;
    __device__ __forceinline__ ProbExp(float m_, ProbFactor f)
        : k(f.k), kl(f.kl), c0(rintf(m_ * f.k * 1024.f) * 0x1p-10f), m(m_), off(1.f), huge(!(fabsf(m_ * f.k) < 4096.f)) {
        if (!huge) off = exp2f(-fmaf(m, kl, fmaf(m, k, -c0)));
    }
    __device__ __forceinline__ float operator()(float x) const {
        if (huge) return ex2(fmaxf((x - m) * k, -200.f));
        const float t = fmaf(x, k, 12582912.f - c0);  // 1.5 2^23: the sum's last bits are n
        const float c = (t - 12582912.f) + c0;
        const float f = fmaf(x, kl, fmaf(x, k, -c));
        const float p = ex2(f);
        return t >= 12582912.f - 126.f ? p * __int_as_float((__float_as_int(t) << 23) + 0x3f800000) : 0.f;
    }
};
// 2^((a - b) k) of two slices' maxima, a <= b, to binary32: an error here is a whole slice's.
__device__ __forceinline__ float prob_scale(float a, float b, ProbFactor f) {
    if (a == b) return 1.f;
    const float d = a - b, bb = d - a, e = (a - (d - bb)) - (b + bb);  // (a - b) - d exactly
    const float h = d * f.k, l = fmaf(d, f.kl, fmaf(e, f.k, fmaf(d, f.k, -h)));
    const float p = exp2f(fmaxf(h, -200.f));
    return fmaf(p, h > -200.f ? l * 0.69314718f : 0.f, p);
}

constexpr int kProbsThreads = 256;
constexpr int kProbsSlice = 16384;  // elements of a row's slice in shared memory

// The row's slices exchange through this (distributed shared memory).
struct ProbsPart {
    float m, s;
    int at;
};

// SM (vocab <= cluster * kProbsSlice): a cluster per row, each CTA a slice in shared memory. The row is
// read once and every exponential formed once: the slice's weights against its own maximum take the
// logits' place, the maxima and sums meet in one exchange, and a product per element is left.
// 320 rows of 128,256: 81 us, 4.0 TB/s, 62 % of a copy's rate (three CTAs an SM start and end with their
// clusters, so loads, exponentials and stores overlap only across clusters; clusters of 16 and CTAs that
// stay for several rows were slower); exponentials took 100 us with the correction at the exponent's size.
// Else (larger vocabularies) a CTA per row reads it three times. VEC: 16-byte aligned rows.
template <bool SM, bool VEC>
__global__ void __launch_bounds__(kProbsThreads) probs_kernel(const ProbsParams p) {
    namespace cg = cooperative_groups;
    extern __shared__ __align__(16) float slice[];
    cg::cluster_group cluster = cg::this_cluster();
    const int C = SM ? (int)cluster.num_blocks() : 1, rank = SM ? (int)cluster.block_rank() : 0;
    const int row = blockIdx.x / C, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    constexpr int NW = kProbsThreads / 32, NT = kProbsThreads;
    __shared__ float red[2][NW];
    __shared__ int redi[NW];
    __shared__ ProbsPart part;
    const int per = SM ? ((p.vocab + C - 1) / C + 3) & ~3 : p.vocab;
    const int v0 = min(p.vocab, rank * per), n = min(p.vocab, v0 + per) - v0;
    const float* x = p.x + (size_t)row * p.ldx + v0;
    float* y = p.y + (size_t)row * p.ldy + v0;
    pdl_wait();
    if constexpr (SM) {
        if constexpr (VEC) {
            for (int i = tid * 4; i + 3 < n; i += NT * 4) cp_async16(slice + i, x + i);
            cp_async_commit();
            if (tid < (n & 3)) slice[(n & ~3) + tid] = x[(n & ~3) + tid];
        } else {
#pragma unroll 4
            for (int i = tid; i < n; i += NT) slice[i] = x[i];
        }
        if ((n & 3) && tid < 4 - (n & 3)) slice[n + tid] = -INFINITY;  // whole groups of four
    }
    const float t = p.temp[row];
    const bool greedy = !(t > 0.f);
    const ProbFactor k(greedy ? 1.f : t);
    if constexpr (SM) {
        if constexpr (VEC) cp_async_wait_all();
        __syncthreads();
    }
    // f(element, its index) over this thread's elements, in ascending order
    auto each = [&](auto&& f) {
        if constexpr (SM) {
#pragma unroll 4
            for (int i = tid * 4; i < n; i += NT * 4) {
                const float4 w = *reinterpret_cast<const float4*>(slice + i);
                f(w.x, i);
                f(w.y, i + 1);
                f(w.z, i + 2);
                f(w.w, i + 3);
            }
        } else {
            for (int i = tid; i < n; i += NT) f(x[i], i);
        }
    };
    float m = -INFINITY, s = 0.f;
    int at = 0x7fffffff;
    each([&](float v, int) { m = fmaxf(m, v); });  // (fmaxf passes a NaN over)
    m = warp_max(m);
    if (lane == 0) red[0][warp] = m;
    __syncthreads();
    m = warp_max(lane < NW ? red[0][lane] : -INFINITY);
    const ProbExp e(m, k);
    if (greedy) {  // the slice's first maximum
        each([&](float v, int i) { if (v == m) at = min(at, i + v0); });
        at = __reduce_min_sync(0xffffffffu, at);
        if (lane == 0) redi[warp] = at;
        __syncthreads();
        at = __reduce_min_sync(0xffffffffu, lane < NW ? redi[lane] : 0x7fffffff);
    } else if (m != -INFINITY) {
        if (m == INFINITY) {
            each([&](float v, int) { s += v == INFINITY ? 1.f : 0.f; });
        } else if constexpr (SM) {  // the weights take the logits' place
            float s4[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
            for (int i = tid * 4; i < n; i += NT * 4) {
                float4 w = *reinterpret_cast<const float4*>(slice + i);
                w.x = e(w.x); w.y = e(w.y); w.z = e(w.z); w.w = e(w.w);
                *reinterpret_cast<float4*>(slice + i) = w;
                s4[0] += w.x; s4[1] += w.y; s4[2] += w.z; s4[3] += w.w;
            }
            s = (s4[0] + s4[1]) + (s4[2] + s4[3]);
        } else {
            each([&](float v, int) { s += e(v); });
        }
        s = warp_sum(s);
        if (lane == 0) red[1][warp] = s;
        __syncthreads();
        s = warp_sum(lane < NW ? red[1][lane] : 0.f);
        if (m != INFINITY) s *= e.off;
    }
    float M = m, S = s;
    if (SM && C > 1) {
        if (tid == 0) part = ProbsPart{m, s, at};
        cluster.sync();
        ProbsPart o{-INFINITY, 0.f, 0x7fffffff};
        if (lane < C) o = *cluster.map_shared_rank(&part, lane);  // every warp for itself
        M = warp_max(o.m);
        S = warp_sum(o.m == -INFINITY || greedy ? 0.f : o.s * prob_scale(o.m, M, k));
        at = __reduce_min_sync(0xffffffffu, o.m == M ? o.at : 0x7fffffff);
        cluster.sync();  // no CTA leaves while another may still read its part
    }
    const float iv = 1.f / S;
    const float part_of = greedy || m == -INFINITY || m == INFINITY ? 0.f : prob_scale(m, M, k) * iv * e.off;
    auto term = [&](float v, int i) {
        if (M == -INFINITY) return 0.f;  // nothing can be chosen
        if (greedy) return i + v0 == at ? 1.f : 0.f;
        if (M == INFINITY) return m == INFINITY && v == INFINITY ? iv : 0.f;  // (a finite slice holds weights)
        if (SM) return m == -INFINITY ? 0.f : v * part_of;  // (a slice of -inf kept its logits)
        return e(v) * part_of;
    };
    if (SM && VEC && !greedy && m != -INFINITY && M != INFINITY) {  // the usual row
#pragma unroll 4
        for (int i = tid * 4; i < n; i += NT * 4) {
            float4 w = *reinterpret_cast<const float4*>(slice + i);
            w.x *= part_of; w.y *= part_of; w.z *= part_of; w.w *= part_of;
            if (i + 3 < n) {
                *reinterpret_cast<float4*>(y + i) = w;
            } else {
                y[i] = w.x;
                if (i + 1 < n) y[i + 1] = w.y;
                if (i + 2 < n) y[i + 2] = w.z;
            }
        }
    } else if constexpr (SM && VEC) {
        for (int i = tid * 4; i < n; i += NT * 4) {
            const float4 w = *reinterpret_cast<const float4*>(slice + i);
            const float4 o = make_float4(term(w.x, i), term(w.y, i + 1), term(w.z, i + 2), term(w.w, i + 3));
            if (i + 3 < n) {
                *reinterpret_cast<float4*>(y + i) = o;
            } else {
                y[i] = o.x;
                if (i + 1 < n) y[i + 1] = o.y;
                if (i + 2 < n) y[i + 2] = o.z;
            }
        }
    } else {
        for (int i = tid; i < n; i += NT) y[i] = term(SM ? slice[i] : x[i], i);
    }
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
constexpr int kVerifyMaxCluster = 8;

__device__ __forceinline__ float prob_in(float x) { return fmaxf(x, 0.f); }  // negative and NaN: 0

// One cluster per sequence. Every CTA finds the first refused token (the numbers are gathered, a
// lane per drafted token), then sums its slice of the row the next token is drawn from, a run of
// consecutive elements per warp; the slices' sums meet in distributed shared memory, and the warp
// whose run holds sample_u * total walks it once more, its CTA's warps together. Sums are in 64 bits:
// 128k binary32 terms in 32 would move the drawn token. 64 sequences of vocabulary 128,256 with a draft's
// probabilities: 17 us for 66 MB, 59 % of a copy's rate; the rest is the chain drafted id -> probability
// -> row -> run and the cluster's meetings. VEC: 16-byte aligned rows.
template <bool VEC>
__global__ void __launch_bounds__(kVerifyThreads, 2) verify_kernel(const VerifyParams p) {
    namespace cg = cooperative_groups;
    cg::cluster_group cluster = cg::this_cluster();
    const int C = (int)cluster.num_blocks(), rank = (int)cluster.block_rank(), s = blockIdx.x / C;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    constexpr int NW = kVerifyThreads / 32;
    __shared__ int s_acc;
    __shared__ double s_sum[2], s_run[NW];
    pdl_wait();
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
                const float u = p.accept_u[(size_t)s * p.max_draft + j];
                refuse = true;
                if (x < (unsigned)p.vocab) {
                    const float pt = prob_in(p.target[((size_t)s * (p.max_draft + 1) + j) * p.ldt + x]);
                    const float qd = p.draft ? prob_in(p.draft[((size_t)s * p.max_draft + j) * p.ldd + x]) : 1.f;
                    // the product of two binary32 numbers is exact in binary64
                    refuse = !((double)u * (double)qd < (double)pt);
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
    auto value = [&](float a, float b, int v) -> double {  // a = P[v], b = Q[v]
        if (mode == 0) return (double)prob_in(a);
        if (Q) return fmax((double)prob_in(a) - (double)prob_in(b), 0.0);
        return (unsigned)v == hole ? 0.0 : (double)prob_in(a);
    };
    // warp w of CTA r: run r * NW + w, a multiple of four elements long
    const int run_len = ((p.vocab + C * NW - 1) / (C * NW) + 3) & ~3;
    const long long first = (long long)(rank * NW + warp) * run_len;
    const int v0 = (int)min((long long)p.vocab, first), v1 = min(p.vocab, v0 + run_len);
    auto four = [&](const float* src, int i, int end, float (&x)[4]) {  // elements i.., zeros from `end` on
        if (VEC && i + 3 < end) {
            *reinterpret_cast<float4*>(x) = *reinterpret_cast<const float4*>(src + i);
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) x[e] = i + e < end ? src[i + e] : 0.f;
        }
    };
    double total = 0.0, before = 0.0;
    int owner = -1;
    for (int pass = 0; pass < 2; ++pass) {
        double a = 0.0, a2 = 0.0;
        const bool sub = mode && Q;
        int i = v0 + lane * 4;
        constexpr int U = 4;  // steps whose loads are in flight together
        for (; VEC && i - lane * 4 + U * 128 <= v1; i += U * 128) {
            float4 x[U], q[U];
#pragma unroll
            for (int u = 0; u < U; ++u) x[u] = __ldcs(reinterpret_cast<const float4*>(P + i + u * 128));
            if (sub) {
#pragma unroll
                for (int u = 0; u < U; ++u) q[u] = __ldcs(reinterpret_cast<const float4*>(Q + i + u * 128));
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const float xs[4] = {x[u].x, x[u].y, x[u].z, x[u].w};
                const float qs[4] = {q[u].x, q[u].y, q[u].z, q[u].w};
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    // (p - q where p > q: exact in 64 bits; NaN compares false)
                    if (sub) {
                        const float qv = prob_in(qs[e]);
                        if (xs[e] > qv) { a += (double)xs[e]; a2 += (double)qv; }
                    } else if (xs[e] > 0.f && (mode == 0 || (unsigned)(i + u * 128 + e) != hole)) {
                        a += (double)xs[e];
                    }
                }
            }
        }
        a -= a2;
        for (; i < v1; i += 128) {
            float x[4], q[4] = {};
            four(P, i, v1, x);
            if (sub) four(Q, i, v1, q);
#pragma unroll
            for (int e = 0; e < 4; ++e) a += value(x[e], q[e], i + e);
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) a += __shfl_xor_sync(0xffffffffu, a, o);
        if (lane == 0) s_run[warp] = a;
        __syncthreads();
        if (warp == 0) {
            double t = lane < NW ? s_run[lane] : 0.0;
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) t += __shfl_xor_sync(0xffffffffu, t, o);
            if (lane == 0) s_sum[pass] = t;
        }
        cluster.sync();
        double part[kVerifyMaxCluster];
        total = 0.0;
#pragma unroll
        for (int j = 0; j < kVerifyMaxCluster; ++j) part[j] = j < C ? *cluster.map_shared_rank(&s_sum[pass], j) : 0.0;
#pragma unroll
        for (int j = 0; j < kVerifyMaxCluster; ++j) total += part[j];
        if (total > 0.0 || mode == 0) {
            const double t = (double)p.sample_u[s] * total;
            double run = 0.0, last_before = 0.0;
            int last = -1;
#pragma unroll
            for (int j = 0; j < kVerifyMaxCluster; ++j) {
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
    // the lowest v of this slice whose running sum exceeds t: every warp finds the run that crosses
    // t (or, where rounding put t at the slice's end, the last with a positive sum), its warp walks it
    const double t = (double)p.sample_u[s] * total - before;
    double base = 0.0, at_base = 0.0;
    int who = -1;
    for (int w = 0; w < NW; ++w) {
        const double a = s_run[w];
        if (a > 0.0) {
            who = w;
            at_base = base;
            if (base + a > t) break;
        }
        base += a;
    }
    if (who < 0) {
        if (tid == 0) out[acc] = 0;  // no positive probability anywhere
        return;
    }
    // the CTA's warps take 128 elements each of that run, 2,048 at a time (one warp alone waited for every
    // load in turn: 29 us on 64 sequences of the 8B vocabulary)
    const long long first_of = (long long)(rank * NW + who) * run_len;
    const int r0 = (int)min((long long)p.vocab, first_of), r1 = min(p.vocab, r0 + run_len);
    __shared__ double s_blk[NW];
    __shared__ int s_hit, s_last;
    if (tid == 0) { s_hit = 0x7fffffff; s_last = r0; }
    double run = at_base;
    for (int i0 = r0; i0 < r1; i0 += NW * 128) {
        const int i = i0 + warp * 128 + lane * 4;
        float x[4] = {}, q[4] = {};
        four(P, i, r1, x);
        if (mode && Q) four(Q, i, r1, q);
        double c[4], mine = 0.0;
        int lastpos = -1;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const double w = i + e < r1 ? value(x[e], q[e], i + e) : 0.0;
            if (w > 0.0) lastpos = i + e;
            mine += w;
            c[e] = mine;
        }
        double incl = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const double u = __shfl_up_sync(0xffffffffu, incl, o);
            if (lane >= o) incl += u;
        }
        __syncthreads();  // (the block before is read)
        if (lane == 31) s_blk[warp] = incl;
        __syncthreads();
        double start = run + (incl - mine);
        for (int w = 0; w < NW; ++w) {
            if (w < warp) start += s_blk[w];
            run += s_blk[w];
        }
        int hit = 0x7fffffff;
#pragma unroll
        for (int e = 3; e >= 0; --e)
            if (i + e < r1 && start + c[e] > t && (e == 0 ? c[0] > 0.0 : c[e] > c[e - 1])) hit = i + e;
        if (hit != 0x7fffffff) atomicMin(&s_hit, hit);
        if (lastpos >= 0) atomicMax(&s_last, lastpos);
        __syncthreads();
        if (s_hit != 0x7fffffff) break;
    }
    if (tid == 0) out[acc] = (unsigned)(s_hit != 0x7fffffff ? s_hit : s_last);
}

}  // namespace laic
