// Attention over a KV cache in pages, with shared prefixes read for all their rows together.
//
// out[r] = sum_t p_t v_t, p = softmax_t(scale q[r] . k_t) over the positions t < n_r of row r's
// sequence. The work is cut into items, each a set of score columns (query row, query head of one
// KV head) over a range of positions:
//   private item: one row's G = heads / kv_heads columns over [shared, n_r): a CTA's four warps where the
//   range is short (it then joins the shared items' results and writes the output), else a warp per split
//   (memory bounds these: 64 rows of up to 8,000 positions, 8 kv heads of 128, 170 us, 6.0 TB/s, 92 % of a
//   copy's rate; a warp's own ring needs no barrier. Its next stage is loaded once the one before it is consumed, so
//   a warp's loads do not run under its own products: the other eight to twelve warps of the SM hide them);
//   shared item (a CTA): up to 8 NT columns (32 at most) of a group's rows over a split of [0, shared), so the keys
//   and values of a shared position are read once for all of them (wide groups: paged_bulk.cuh, up to 256 columns at
//   once; more columns, and at head_dim 32 more than 32, read them again, mostly out of L2). What bounds
//   them is each warp's chain load -> QK -> softmax -> PV, so CTAs per SM count: eight groups of five rows,
//   20 columns of head_dim 64, 500 to 8,000 positions take 33 us with four CTAs an SM, 45 with three.
// An item keeps, per column, a reference m (a maximum of the scores seen, log2 domain, renewed when
// they outgrow it by 2^8), l = sum 2^(s - m) and the unnormalised output; where a row has several
// items the merge kernel joins them by out = sum_i o_i 2^(m_i - M) / sum_i l_i 2^(m_i - M).
//
// Products run transposed on mma.m16n8k16: S^T = K Q^T (16 positions x 8 columns) and
// O^T = V^T P^T, so the few columns of a decode step fill the narrow side of the tile; P^T goes
// from accumulators to B fragments by movmatrix. FP32 queries and weights are split into binary16
// hi + lo (two products, 22 bits); a query row is first scaled by a power of two to [1, 2), so no
// magnitude leaves binary16's range, and the weights carry a factor 2^7 that keeps small ones
// out of its subnormals (both sides of the final division have it, and 2^8 2^7 stay below its largest).
// The hi and lo products have accumulators of their own: the tensor cores truncate as they accumulate, and lo parts added to a
// large sum would only lengthen that chain. A private item of at most four columns (a decode step of
// the usual groups) has hi and lo side by side in one tile's eight columns (PK), so the split costs no
// product at all.
#pragma once
#include "common.cuh"
#include "mma_matvec.cuh"  // smem_u32, mma16816, cp.async
#include "attention.cuh"   // attn_swz, ldsm_x4
#include "paged.cuh"

namespace laic {

struct KvAttnParams {
    const void* q;
    void* out;
    long long ldq, ldo;
    const __half *kp, *vp;
    int num_pages, page_shift, kv_heads, heads, G;
    const int *len, *seq, *table;
    int nseq, pages_per_seq, rows, max_len;
    int groups, max_group_rows, max_shared, max_private;
    const int *group_rows, *group_len;
    float scale_log2;             // scale * log2(e)
    int lp, nsp;                  // private splits: positions each, count
    int ls, nss, ctiles;          // shared splits, column tiles per group
    int lc;                       // splits joined into one partial (the bulk kernel's clusters; else 1)
    int private_items;
    bool q_vec, out_vec;          // rows of q, of out are 16-byte aligned
    uint32_t g_inv;               // 2^16 / G rounded up
    float* part_o;                // [rows][heads][nss + nsp][head_dim]
    float2* part_ml;              // [rows][heads][nss + nsp] (m, l)
    int first;                    // private items: no kernel of this call before them
    int direct;                   // the bulk kernel's clusters hold all that their rows see: they write the output
    int* err;
};

constexpr int kPaWarps = 4;
constexpr int kPaChunk = 64;      // positions per ring stage: 16 per warp
constexpr int kPaMaxSplit = 2048; // positions per item at most (its page ids are held in shared memory)
constexpr float kPaSlack = 8.f;  // log2 of how far a maximum may outgrow its reference before sums are rescaled
constexpr float kPaGain = 128.f;  // the factor the weights carry (bulk items too: a row's items are summed)

__host__ __device__ constexpr int pa_stages(int D) { (void)D; return 3; }
__host__ __device__ constexpr size_t pa_ring_bytes(int D) { return (size_t)pa_stages(D) * 2 * kPaChunk * D * 2; }
__host__ __device__ constexpr size_t pa_smem(int D, int NT, bool hl) {
    const size_t ring = pa_ring_bytes(D), red = (size_t)kPaWarps * NT * 8 * (D + 4) * 4;
    return (ring > red ? ring : red) + (size_t)(D / 16) * NT * (hl ? 2 : 1) * 32 * 8;
}

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ uint32_t movm_t(uint32_t a) {
    uint32_t d;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
    return d;
}
// 16 bytes, or 16 zeros where !live (the source is not read then).
__device__ __forceinline__ void cp_async16_z(uint32_t dst, const void* src, bool live) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(live ? 16 : 0) : "memory");
}
template <int N>
__device__ __forceinline__ void cp_async_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// What the index arrays say about one row.
struct RowView {
    int n;       // positions seen (0: none); -1: padding
    int shared;  // of those, the group's
    int seq;
};
__host__ __device__ inline int kv_clamp_len(const KvAttnParams& p, int n, int bound) {
    const int most = p.pages_per_seq << p.page_shift, cap = bound < most ? bound : most;
    if (n > cap) {
        kv_flag(p.err, kKvBadPos);
        n = cap;
    }
    return n;
}
// Rows [r0, r1) of group g, false (and recorded) where they are not within the call's rows and bounds.
__host__ __device__ inline bool group_rows(const KvAttnParams& p, int g, int& r0, int& r1) {
    r0 = p.group_rows[g];
    r1 = p.group_rows[g + 1];
    if (r0 < 0 || r1 < r0 || r1 > p.rows || r1 - r0 > p.max_group_rows) {
        kv_flag(p.err, kKvBadGroup);
        return false;
    }
    return true;
}
// Length and sequence of row r.
struct RowAt {
    int n, seq;
};
__host__ __device__ inline RowAt row_at(const KvAttnParams& p, int r) { return RowAt{p.len[r], p.seq ? p.seq[r] : r}; }
// The page table row through which the group of rows [r0, r1) is read: that of its first row that sees any
// position (padding may name any sequence, and one that sees nothing need hold nothing). A bad one is recorded, and
// reads some sequence's pages. `lead`: row r0, which the caller loads while other loads are under way.
__host__ __device__ inline int group_seq(const KvAttnParams& p, int r0, int r1, RowAt lead) {
    for (int r = r0 + 1; lead.n <= 0 && r < r1; ++r) lead = row_at(p, r);
    if (lead.n <= 0) return 0;  // nothing is read
    if (lead.seq >= 0 && lead.seq < p.nseq) return lead.seq;
    kv_flag(p.err, kKvBadSeq);
    return 0;
}
// Shared positions of group g.
__host__ __device__ inline int group_shared(const KvAttnParams& p, int g) {
    const int n = kv_clamp_len(p, p.group_len[g], p.max_shared);
    return n > 0 ? n : 0;
}
// The shared length of row r's group: `n` threads tid of one sync domain search together and leave it
// in *found (reset to 0 before, synchronised after, by the caller).
__device__ __forceinline__ void find_group(const KvAttnParams& p, int r, int tid, int n, int* found) {
    for (int g = tid; g < p.groups; g += n) {
        int r0, r1;
        if (group_rows(p, g, r0, r1) && r >= r0 && r < r1) *found = group_shared(p, g);
    }
}
__host__ __device__ inline RowView row_view(const KvAttnParams& p, int n, int s, int shared) {  // n, s: len[r], seq[r]
    RowView v;
    v.n = -1;
    v.seq = -1;
    v.shared = 0;
    if (n < 0) return v;
    v.n = kv_clamp_len(p, n, p.max_len);
    if (s >= 0 && s < p.nseq) {
        v.seq = s;
    } else {
        kv_flag(p.err, kKvBadSeq);
        v.n = 0;
    }
    v.shared = v.n < shared ? v.n : shared;
    return v;
}
__host__ __device__ inline RowView row_view(const KvAttnParams& p, int r, int shared) {
    return row_view(p, p.len[r], p.seq ? p.seq[r] : r, shared);
}

// The maximum that an item reports beside its sum: a column all of whose scores are NaN has none, but its sum (NaN)
// has to reach the row.
__device__ __forceinline__ float seen_max(float m, float sum) { return m == -INFINITY && sum != sum ? 0.f : m; }

// A value that is not finite reaches the rows that see it whatever its weight. The products may make NaN of an
// infinite one (a weight rounded to zero, its lo part's zero or sign, an item's weight in a join), so where an output
// is NaN and the sum of its weights is not, it is the sum of the values of its dimension d that are not finite, over
// the positions that row r sees; x where there is none. Outputs are looked up once they are stored: the usual call
// pays for one test per output.
__device__ __forceinline__ float odd_output(const KvAttnParams& p, int r, int kvh, int D, int d, float x) {
    int shared = 0, lead = 0;
    for (int g = 0; g < p.groups; ++g) {
        int r0, r1;
        if (!group_rows(p, g, r0, r1) || r < r0 || r >= r1) continue;
        shared = group_shared(p, g);
        lead = group_seq(p, r0, r1, row_at(p, r0));
    }
    const RowView v = row_view(p, r, shared);
    const int end = min(v.n, v.shared + p.max_private);
    float sum = 0.f;
    bool any = false;
#pragma unroll 1
    for (int t0 = 0; t0 < end; t0 += 8) {  // (8 positions lie in one page)
        auto page_of = [&](int seq) {
            const int id = p.table[(size_t)max(0, seq) * p.pages_per_seq + (t0 >> p.page_shift)];
            return id >= 0 && id < p.num_pages ? id : 0;
        };
        const int common = page_of(lead), own = page_of(v.seq);
        float y[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int t = t0 + i, page = t < v.shared ? common : own;
            y[i] = t < end ? __half2float(p.vp[((((size_t)page * p.kv_heads + kvh) << p.page_shift) + (t & ((1 << p.page_shift) - 1))) * D + d])
                           : 0.f;
        }
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (!(fabsf(y[i]) <= 65504.f)) {
                sum += y[i];
                any = true;
            }
    }
    return any ? sum : x;
}
template <typename T>
__device__ __forceinline__ void odd_outputs(const KvAttnParams& p, int r, int kvh, int D, int d, T* stored, int n) {
#pragma unroll 1
    for (int k = 0; k < n; ++k) {
        const float x = kv_in<T>(stored[k]);
        if (x != x) stored[k] = kv_out<T>(odd_output(p, r, kvh, D, d + k, x));
    }
}

// Elements e and e + 1 (e even) of query row r.
template <typename T>
__device__ __forceinline__ float2 q_pair(const KvAttnParams& p, int r, int e) {
    const T* q = static_cast<const T*>(p.q) + (size_t)r * p.ldq + e;
    if (!p.q_vec) return make_float2(kv_in<T>(q[0]), kv_in<T>(q[1]));
    if constexpr (sizeof(T) == 4) return *reinterpret_cast<const float2*>(q);
    else return __half22float2(*reinterpret_cast<const __half2*>(q));
}

// One item: columns [col0, col0 + 8 NT) of rows r0.. (column = row offset * G + head), positions
// [t0, t1) of sequence `seq`. Column c sees positions below lim[c] (shared memory; 0: no column).
// slot: the partial's index among its row's; minlim: the smallest lim of a live column.
template <int D, int NT, typename T>
__device__ __forceinline__ void pa_item(const KvAttnParams& p, int r0, int col0, int ncol, int kvh, int seq, int t0,
                                        int t1, int slot, const int* lim, int minlim, int* page_ids, float* cmul,
                                        uint8_t* smem) {
    constexpr bool HL = sizeof(T) == 4;  // a second set of products for the lo parts
    constexpr int HN = HL ? 2 : 1;
    constexpr int KS = D / 16, CPR = D / 8, NC = NT * 8, NW = kPaWarps, NTH = kPaWarps * 32;
    constexpr int NST = pa_stages(D);
    constexpr size_t kRed = (size_t)NW * NC * (D + 4) * 4;
    constexpr size_t kQoff = pa_ring_bytes(D) > kRed ? pa_ring_bytes(D) : kRed;
    uint32_t* qf = reinterpret_cast<uint32_t*>(smem + kQoff);  // [KS][NT][HN][32 lanes][2]
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int gq = lane >> 2, c = lane & 3;

    // ---- the range's page ids, each checked once
    const int first_page = t0 >> p.page_shift;
    const int npages = t1 > t0 ? ((t1 - 1) >> p.page_shift) - first_page + 1 : 0;
    for (int i = tid; i < npages; i += NTH) {
        int id = p.table[(size_t)seq * p.pages_per_seq + first_page + i];
        if (id < 0 || id >= p.num_pages) {
            kv_flag(p.err, kKvBadPage);
            id = 0;
        }
        page_ids[i] = id;
    }
    __syncthreads();

    // chunks start at a multiple of 16, so that 16 positions lie in one page (positions before t0 are masked)
    const int a0 = t0 & ~15;
    const int nch = (t1 - a0 + kPaChunk - 1) / kPaChunk;
    const uint32_t ring = smem_u32(smem);
    constexpr uint32_t STAGE = 2 * kPaChunk * D * 2;
    constexpr int RPP = NTH / CPR;  // rows a pass of the CTA covers; a thread's row within 8 stays the same
    const int lrow = tid / CPR, lcc = tid % CPR;
    const uint32_t dst0 = ring + 2 * attn_swz<D>(lrow, lcc);
    const size_t src0 = (size_t)(lrow & 15) * D + lcc * 8;
    const int page_mask = (1 << p.page_shift) - 1;
    auto load = [&](int ch) {
        if (ch < nch) {
            const int c0 = a0 + ch * kPaChunk;
            const uint32_t kd = dst0 + (uint32_t)(ch % NST) * STAGE;
            size_t off = 0;
#pragma unroll
            for (int i = 0; i < kPaChunk / RPP; ++i) {
                const int r = lrow + i * RPP;
                if (RPP >= 16 || i % (16 / RPP) == 0) {  // a new block of 16 positions
                    const int tb = c0 + (r & ~15);
                    const int page = tb < t1 ? page_ids[(tb >> p.page_shift) - first_page] : 0;
                    off = ((((size_t)page * p.kv_heads + kvh) << p.page_shift) + (tb & page_mask)) * D + src0;
                }
                const size_t at = off + (RPP < 16 ? (i % (16 / RPP)) * RPP * D : 0);
                const bool live = c0 + r < t1;  // rows past the end: zeros
                cp_async16_z(kd + i * RPP * D * 2, p.kp + at, live);
                cp_async16_z(kd + kPaChunk * D * 2 + i * RPP * D * 2, p.vp + at, live);
            }
        }
        cp_async_commit();
    };
#pragma unroll
    for (int s = 0; s < NST - 1; ++s) load(s);

    // ---- query fragments: a warp per column
    for (int col = warp; col < NC; col += NW) {
        const int cc = col0 + col;
        const bool live = cc < ncol;
        const int rr = r0 + (live ? cc / p.G : 0), hh = (kvh * p.G + (live ? cc % p.G : 0)) * D;
        constexpr int PL = (D / 2 + 31) / 32;  // pairs per lane
        float a[PL], b[PL], mx = 0.f;
#pragma unroll
        for (int i = 0; i < PL; ++i) {
            const int pi = lane + 32 * i;
            const bool in = live && pi < D / 2;
            const float2 x = in ? q_pair<T>(p, rr, hh + 2 * pi) : make_float2(0.f, 0.f);
            a[i] = x.x;
            b[i] = x.y;
            mx = fmaxf(mx, fmaxf(fabsf(a[i]), fabsf(b[i])));
        }
        float fac = 1.f, inv = 1.f;
        if (HL) {
            mx = warp_max(mx);
            const int e = min(max((int)(__float_as_uint(mx) >> 23) - 127, -100), 120);
            fac = __uint_as_float((uint32_t)(127 - e) << 23);
            inv = __uint_as_float((uint32_t)(127 + e) << 23);
        }
        if (lane == 0) cmul[col] = p.scale_log2 * inv;
#pragma unroll
        for (int i = 0; i < PL; ++i) {
            const int pi = lane + 32 * i;
            if (pi < D / 2) {
                const int ks = pi >> 3, j = (pi >> 2) & 1, cl = pi & 3;
                uint32_t* dst = qf + (((size_t)(ks * NT + (col >> 3)) * HN) * 32 + (col & 7) * 4 + cl) * 2 + j;
                const float va = a[i] * fac, vb = b[i] * fac;
                const __half ha = __float2half_rn(va), hb = __float2half_rn(vb);
                dst[0] = pack_h2(ha, hb);
                if (HL) dst[64] = pack_h2(__float2half_rn(va - __half2float(ha)), __float2half_rn(vb - __half2float(hb)));
            }
        }
    }

    float m_[NT][2], l_[NT][2], o[KS][NT][4];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
        m_[nt][0] = m_[nt][1] = -INFINITY;
        l_[nt][0] = l_[nt][1] = 0.f;
#pragma unroll
        for (int mt = 0; mt < KS; ++mt) o[mt][nt][0] = o[mt][nt][1] = o[mt][nt][2] = o[mt][nt][3] = 0.f;
    }
    const int li = lane >> 3, lr = lane & 7;  // ldmatrix: this lane addresses row lr of matrix li
    const int wp = warp * 16;                 // this warp's first position of a chunk

    uint2 qr[NT == 1 ? KS : 1][HN];  // one tile: the query fragments stay in registers
    for (int ch = 0; ch < nch; ++ch) {
        cp_async_wait<NST - 2>();
        __syncthreads();  // chunk ch is in shared memory, and chunk ch - 1 consumed
        if (NT == 1 && ch == 0) {
#pragma unroll
            for (int ks = 0; ks < KS; ++ks)
#pragma unroll
                for (int hl = 0; hl < HN; ++hl) qr[ks][hl] = *reinterpret_cast<const uint2*>(qf + ((ks * HN + hl) * 32 + lane) * 2);
        }
        load(ch + NST - 1);
        const int c0 = a0 + ch * kPaChunk;
        if (c0 + wp < t1 && c0 + wp + 16 > t0) {
            const uint32_t ks_a = ring + (uint32_t)(ch % NST) * (2 * kPaChunk * D * 2), vs_a = ks_a + kPaChunk * D * 2;
            float s[NT][4], sl[NT][4];
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                s[nt][0] = s[nt][1] = s[nt][2] = s[nt][3] = 0.f;
                sl[nt][0] = sl[nt][1] = sl[nt][2] = sl[nt][3] = 0.f;
            }
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) {
                uint32_t a[4];
                ldsm_x4(ks_a + 2 * attn_swz<D>(wp + (li & 1) * 8 + lr, ks * 2 + (li >> 1)), a);
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                    const uint32_t* qa = qf + (((ks * NT + nt) * HN) * 32 + lane) * 2;
                    const uint2 b = NT == 1 ? qr[NT == 1 ? ks : 0][0] : *reinterpret_cast<const uint2*>(qa);
                    mma16816_acc(s[nt], a[0], a[1], a[2], a[3], b.x, b.y);
                    if (HL) {
                        const uint2 bl = NT == 1 ? qr[NT == 1 ? ks : 0][HN - 1] : *reinterpret_cast<const uint2*>(qa + 64);
                        mma16816_acc(sl[nt], a[0], a[1], a[2], a[3], bl.x, bl.y);
                    }
                }
            }
            const int pos = c0 + wp + gq;
            const bool full = c0 + wp >= t0 && c0 + wp + 16 <= min(t1, minlim);  // every live column sees all 16 positions
            uint32_t ph[NT][2], pl[NT][2];
            float cm2[NT][2], mx[NT][2];
            int lm[NT][2];
            bool grew = false;
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const int col = nt * 8 + 2 * c + h;
                    cm2[nt][h] = cmul[col];
                    lm[nt][h] = min(t1, lim[col]);
                    mx[nt][h] = -INFINITY;
                }
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    if (HL) s[nt][e] += sl[nt][e];
                    const float x = s[nt][e] * cm2[nt][e & 1];
                    const int at = pos + (e >> 1) * 8;
                    if (full || (at < lm[nt][e & 1] && at >= t0)) mx[nt][e & 1] = fmaxf(mx[nt][e & 1], x);
                }
                grew |= mx[nt][0] > m_[nt][0] + kPaSlack || mx[nt][1] > m_[nt][1] + kPaSlack;
            }
            if (__any_sync(0xffffffffu, grew)) {  // new reference maxima
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                    float corr[2];
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        float x = mx[nt][h];
                        x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 4));
                        x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 8));
                        x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 16));
                        const float mnew = fmaxf(m_[nt][h], x);
                        corr[h] = mnew == -INFINITY ? 1.f : ex2(m_[nt][h] - mnew);
                        m_[nt][h] = mnew;
                        l_[nt][h] *= corr[h];
                    }
#pragma unroll
                    for (int mt = 0; mt < KS; ++mt) {
                        o[mt][nt][0] *= corr[0]; o[mt][nt][1] *= corr[1];
                        o[mt][nt][2] *= corr[0]; o[mt][nt][3] *= corr[1];
                    }
                }
            }
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
                for (int h = 0; h < 2; ++h) mx[nt][h] = m_[nt][h] == -INFINITY ? 0.f : m_[nt][h];  // (nothing seen yet)
                float pv[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    pv[e] = ex2(fmaf(s[nt][e], cm2[nt][e & 1], -mx[nt][e & 1]));
                    const int at = pos + (e >> 1) * 8;
                    if (!full && (at >= lm[nt][e & 1] || at < t0)) pv[e] = 0.f;
                    l_[nt][e & 1] += pv[e];  // this lane's positions
                    pv[e] *= kPaGain;
                }
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    const __half h0 = __float2half_rn(pv[2 * j]), h1 = __float2half_rn(pv[2 * j + 1]);
                    if (HL)
                        pl[nt][j] = movm_t(pack_h2(__float2half_rn(pv[2 * j] - __half2float(h0)),
                                                   __float2half_rn(pv[2 * j + 1] - __half2float(h1))));
                    ph[nt][j] = movm_t(pack_h2(h0, h1));
                }
#pragma unroll
                for (int e = 0; e < 4; ++e) s[nt][e] = pv[e];
            }
            // a position that some columns see and others do not: where its value is not finite,
            // 0 * inf would reach the others, so those products are summed one by one
            bool odd = false;
            if (!full && min(c0 + wp + 16, t1) > minlim) {  // (positions before t0 are seen too, by other items)
#pragma unroll
                for (int i = lane; i < 16 * CPR; i += 32) {
                    const uint4 w = lds128(vs_a + 2 * attn_swz<D>(wp + i / CPR, i % CPR));
                    const uint32_t x[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
                    for (int k = 0; k < 4; ++k)
                        odd |= (x[k] & 0x7c00u) == 0x7c00u || (x[k] & 0x7c000000u) == 0x7c000000u;
                }
                odd = __any_sync(0xffffffffu, odd);
            }
            if (!odd) {
#pragma unroll
                for (int mt = 0; mt < KS; ++mt) {
                    uint32_t a[4];
                    ldsm_x4_t(vs_a + 2 * attn_swz<D>(wp + (li >> 1) * 8 + lr, mt * 2 + (li & 1)), a);
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) {
                        mma16816_acc(o[mt][nt], a[0], a[1], a[2], a[3], ph[nt][0], ph[nt][1]);
                        if (HL) mma16816_acc(o[mt][nt], a[0], a[1], a[2], a[3], pl[nt][0], pl[nt][1]);
                    }
                }
            } else {
                const __half* V = reinterpret_cast<const __half*>(smem + (size_t)(ch % NST) * (2 * kPaChunk * D * 2) +
                                                                  kPaChunk * D * 2);
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {  // (a weight that is seen is not zero)
                        const int at = pos + (e >> 1) * 8;
                        if (at < lm[nt][e & 1] && at >= t0) s[nt][e] = fmaxf(s[nt][e], 0x1p-126f);
                    }
#pragma unroll 1
                for (int i = 0; i < 16; ++i) {
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                        for (int h = 0; h < 2; ++h) {  // the weight of (position i, column 2c + h): lane (i % 8, c)
                            const float w0 = __shfl_sync(0xffffffffu, s[nt][h], (i & 7) * 4 + c);
                            const float w1 = __shfl_sync(0xffffffffu, s[nt][2 + h], (i & 7) * 4 + c);
                            const float w = i < 8 ? w0 : w1;
                            if (w != 0.f) {
#pragma unroll
                                for (int mt = 0; mt < KS; ++mt)
#pragma unroll
                                    for (int k = 0; k < 2; ++k) {
                                        const int d = mt * 16 + gq + 8 * k;
                                        const float x = __half2float(V[attn_swz<D>(wp + i, d >> 3) + (d & 7)]);
                                        o[mt][nt][2 * k + h] = fmaf(w, x, o[mt][nt][2 * k + h]);
                                    }
                            }
                        }
                }
            }
        }
    }
    cp_async_wait<0>();
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            float v = l_[nt][h];
            v += __shfl_xor_sync(0xffffffffu, v, 4);
            v += __shfl_xor_sync(0xffffffffu, v, 8);
            v += __shfl_xor_sync(0xffffffffu, v, 16);
            l_[nt][h] = v * kPaGain;
            m_[nt][h] = seen_max(m_[nt][h], v);
        }

    // ---- join the warps (the ring holds their outputs now)
    __shared__ float cm[kPaWarps][NC], cl[kPaWarps][NC];
    __syncthreads();
    float* red = reinterpret_cast<float*>(smem);  // [warp][column][D + 4]
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
        if (gq == 0) {
            cm[warp][nt * 8 + 2 * c] = m_[nt][0]; cm[warp][nt * 8 + 2 * c + 1] = m_[nt][1];
            cl[warp][nt * 8 + 2 * c] = l_[nt][0]; cl[warp][nt * 8 + 2 * c + 1] = l_[nt][1];
        }
#pragma unroll
        for (int mt = 0; mt < KS; ++mt)
#pragma unroll
            for (int e = 0; e < 4; ++e)
                red[((size_t)warp * NC + nt * 8 + 2 * c + (e & 1)) * (D + 4) + mt * 16 + gq + (e >> 1) * 8] = o[mt][nt][e];
    }
    __syncthreads();
    const int ns = p.nss + p.nsp;
    for (int i = tid; i < NC * (D / 4); i += NTH) {
        const int col = i / (D / 4), d = (i % (D / 4)) * 4, cc = col0 + col;
        if (cc >= ncol) continue;
        float M = -INFINITY, L = 0.f, w[NW];
#pragma unroll
        for (int k = 0; k < NW; ++k) M = fmaxf(M, cm[k][col]);
        float4 A = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int k = 0; k < NW; ++k) {
            w[k] = cm[k][col] == -INFINITY ? 0.f : ex2(cm[k][col] - M);
            L = fmaf(cl[k][col], w[k], L);
            if (cm[k][col] != -INFINITY) {
                const float4 v = *reinterpret_cast<const float4*>(red + ((size_t)k * NC + col) * (D + 4) + d);
                A.x = fmaf(v.x, w[k], A.x); A.y = fmaf(v.y, w[k], A.y);
                A.z = fmaf(v.z, w[k], A.z); A.w = fmaf(v.w, w[k], A.w);
            }
        }
        const int r = r0 + cc / p.G, h = kvh * p.G + cc % p.G;
        const size_t at = ((size_t)r * p.heads + h) * ns + slot;
        *reinterpret_cast<float4*>(p.part_o + at * D + d) = A;
        if (d == 0) p.part_ml[at] = make_float2(M, L);
    }
}

constexpr int kPrWarps = 4;
// 16 positions of K and V each, per warp (three: fewer CTAs per SM, 173.8 us against 172.4 for 64 rows of 1,024 to
// 8,192 positions, 8 kv heads of 128, though 39.7 against 41.0 for 64 rows of up to 512 behind a shared prefix)
constexpr int kPrStages = 2;
constexpr int kPrWhole = 1024;    // no split is longer, and no range that stays whole
__host__ __device__ constexpr size_t pr_smem(int D) { return (size_t)kPrWarps * kPrStages * 2 * 16 * D * 2; }

// One row's own positions, every warp on its own ring of 16-position stages.
// WHOLE: a CTA per [row][kv head], its warps take turns at the blocks of 16 positions; at the end they
// and the row's shared items (the kernel before this one) are joined and the output written.
// Else: a warp per item of [row][kv head][split], no barrier between the warps.
// PK: FP32 rows of at most four columns, hi parts in columns 0-3, lo parts in 4-7 of the tile.
template <int D, typename T, bool PK, bool WHOLE>
__global__ void __launch_bounds__(kPrWarps * 32) paged_private_kernel(const KvAttnParams p) {
    constexpr int NW = kPrWarps;
    constexpr bool HL = sizeof(T) == 4 && !PK;
    constexpr int HN = HL ? 2 : 1, KS = D / 16, CPR = D / 8, NST = kPrStages;
    constexpr uint32_t STAGE = 2 * 16 * D * 2;
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ int page_ids[NW][kPrWhole / 16 + 2];
    __shared__ uint32_t qf[NW][KS][HN][32][2];
    __shared__ float cmul[NW][8];
    __shared__ int found[NW];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int gq = lane >> 2, c = lane & 3;
    if (p.first) pdl_wait();  // what the stream held before this call
    pdl_launch_dependents();  // (the merge waits for this grid's end; nothing else follows)
    int i = WHOLE ? blockIdx.x : blockIdx.x * NW + warp;
    const bool in = WHOLE || i < p.private_items;
    if (!in) i = 0;
    const int split = WHOLE ? 0 : i % p.nsp;
    if (!WHOLE) i /= p.nsp;
    const int kvh = i % p.kv_heads, r = i / p.kv_heads;
    const int len = p.len[r], sq = p.seq ? p.seq[r] : r;  // under way while the groups are searched
    int shared = 0;
    if (p.groups) {
        if (lane == 0) found[warp] = 0;
        __syncwarp();
        find_group(p, r, lane, 32, &found[warp]);
        __syncwarp();
        shared = found[warp];
    }
    const RowView v = row_view(p, len, sq, shared);
    if (v.n - v.shared > p.max_private && lane == 0) kv_flag(p.err, kKvBadPos);
    if (WHOLE && v.n < 0) {  // padding
        if (blockIdx.x == 0) pdl_wait();
        return;
    }
    const int t0 = v.shared + split * p.lp, t1 = in ? min(min(v.n, v.shared + p.max_private), t0 + p.lp) : 0;
    constexpr int STRIDE = WHOLE ? NW : 1;
    const int a0 = t0 & ~15, first = WHOLE ? warp : 0;  // blocks first, first + STRIDE, ... of 16 positions from a0
    const int nb = in && v.n >= 0 && t0 < t1 ? (((t1 - a0 + 15) >> 4) - first + STRIDE - 1) / STRIDE : 0;
    float m_[2] = {-INFINITY, -INFINITY}, l_[2] = {0.f, 0.f}, o[KS][4];
#pragma unroll
    for (int mt = 0; mt < KS; ++mt) o[mt][0] = o[mt][1] = o[mt][2] = o[mt][3] = 0.f;
    if (nb > 0) {
        // ---- the range's page ids, each checked once; blocks of 16 positions lie in one page
        const int first_page = a0 >> p.page_shift, npages = ((t1 - 1) >> p.page_shift) - first_page + 1;
        for (int k = lane; k < npages; k += 32) {
            int id = p.table[(size_t)v.seq * p.pages_per_seq + first_page + k];
            if (id < 0 || id >= p.num_pages) {
                kv_flag(p.err, kKvBadPage);
                id = 0;
            }
            page_ids[warp][k] = id;
        }
        __syncwarp();
        const uint32_t ring = smem_u32(smem) + (uint32_t)warp * (NST * STAGE);
        constexpr int RPP = 32 / CPR;  // rows a pass of the warp covers
        const int lrow = lane / CPR, lcc = lane % CPR;
        const int page_mask = (1 << p.page_shift) - 1;
        const size_t src0 = (size_t)lrow * D + lcc * 8;
        auto load = [&](int b) {
            if (b < nb) {
                const int tb = a0 + (first + b * STRIDE) * 16;
                const size_t at = ((((size_t)page_ids[warp][(tb >> p.page_shift) - first_page] * p.kv_heads + kvh) << p.page_shift) +
                                   (tb & page_mask)) * D + src0;
                const uint32_t kd = ring + (uint32_t)(b % NST) * STAGE;
#pragma unroll
                for (int q = 0; q < 16 / RPP; ++q) {
                    const int rr = lrow + q * RPP;
                    const bool ok = tb + rr < t1;  // rows past the end: zeros
                    cp_async16_z(kd + 2 * attn_swz<D>(rr, lcc), p.kp + at + (size_t)q * RPP * D, ok);
                    cp_async16_z(kd + 16 * D * 2 + 2 * attn_swz<D>(rr, lcc), p.vp + at + (size_t)q * RPP * D, ok);
                }
            }
            cp_async_commit();
        };
#pragma unroll
        for (int b = 0; b < NST - 1; ++b) load(b);

        // ---- query fragments, column by column
        constexpr int PL = (D / 2 + 31) / 32;  // pairs per lane
        float qa[8][PL][2];
#pragma unroll
        for (int col = 0; col < (PK ? 4 : 8); ++col)
#pragma unroll
            for (int k = 0; k < PL; ++k) {
                const int pi = lane + 32 * k, hh = (kvh * p.G + col) * D;
                const bool got = col < p.G && pi < D / 2;
                const float2 x = got ? q_pair<T>(p, r, hh + 2 * pi) : make_float2(0.f, 0.f);
                qa[col][k][0] = x.x;
                qa[col][k][1] = x.y;
            }
#pragma unroll
        for (int col = 0; col < (PK ? 4 : 8); ++col) {
            float fac = 1.f, inv = 1.f;
            if (HL || PK) {
                float mx = 0.f;
#pragma unroll
                for (int k = 0; k < PL; ++k) mx = fmaxf(mx, fmaxf(fabsf(qa[col][k][0]), fabsf(qa[col][k][1])));
                mx = warp_max(mx);
                const int e = min(max((int)(__float_as_uint(mx) >> 23) - 127, -100), 120);
                fac = __uint_as_float((uint32_t)(127 - e) << 23);
                inv = __uint_as_float((uint32_t)(127 + e) << 23);
            }
            if (lane == 0) cmul[warp][col] = p.scale_log2 * inv;
#pragma unroll
            for (int k = 0; k < PL; ++k) {
                const int pi = lane + 32 * k;
                if (pi < D / 2) {
                    const int ks = pi >> 3, j = (pi >> 2) & 1, cl = pi & 3;
                    const float va = qa[col][k][0] * fac, vb = qa[col][k][1] * fac;
                    const __half ha = __float2half_rn(va), hb = __float2half_rn(vb);
                    qf[warp][ks][0][col * 4 + cl][j] = pack_h2(ha, hb);
                    if (HL || PK) {
                        const uint32_t lo = pack_h2(__float2half_rn(va - __half2float(ha)), __float2half_rn(vb - __half2float(hb)));
                        if (HL) qf[warp][ks][HN - 1][col * 4 + cl][j] = lo;
                        else qf[warp][ks][0][(col + 4) * 4 + cl][j] = lo;
                    }
                }
            }
        }
        __syncwarp();
        uint2 qr[KS][HN];
#pragma unroll
        for (int ks = 0; ks < KS; ++ks)
#pragma unroll
            for (int hl = 0; hl < HN; ++hl) qr[ks][hl] = *reinterpret_cast<const uint2*>(qf[warp][ks][hl][lane]);
        const float cm2[2] = {cmul[warp][PK ? (2 * c) & 3 : 2 * c], cmul[warp][PK ? (2 * c + 1) & 3 : 2 * c + 1]};

        const int li = lane >> 3, lr = lane & 7;  // ldmatrix: this lane addresses row lr of matrix li
        for (int b = 0; b < nb; ++b) {
            cp_async_wait<NST - 2>();
            __syncwarp();
            const uint32_t ks_a = ring + (uint32_t)(b % NST) * STAGE, vs_a = ks_a + 16 * D * 2;
            float s[4] = {0.f, 0.f, 0.f, 0.f}, s2[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) {
                uint32_t a[4];
                ldsm_x4(ks_a + 2 * attn_swz<D>((li & 1) * 8 + lr, ks * 2 + (li >> 1)), a);
                // (two accumulators: the second takes the lo parts, or every other step)
                if (HL) {
                    mma16816_acc(s, a[0], a[1], a[2], a[3], qr[ks][0].x, qr[ks][0].y);
                    mma16816_acc(s2, a[0], a[1], a[2], a[3], qr[ks][HN - 1].x, qr[ks][HN - 1].y);
                } else if (ks & 1) {
                    mma16816_acc(s2, a[0], a[1], a[2], a[3], qr[ks][0].x, qr[ks][0].y);
                } else {
                    mma16816_acc(s, a[0], a[1], a[2], a[3], qr[ks][0].x, qr[ks][0].y);
                }
            }
            const int c0 = a0 + (first + b * STRIDE) * 16, pos = c0 + gq;
            const bool full = c0 >= t0 && c0 + 16 <= t1;
            float mx[2] = {-INFINITY, -INFINITY}, pv[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                s[e] += s2[e];
                if (PK) s[e] += __shfl_xor_sync(0xffffffffu, s[e], 2);
                const int at = pos + (e >> 1) * 8;
                if (full || (at >= t0 && at < t1)) mx[e & 1] = fmaxf(mx[e & 1], s[e] * cm2[e & 1]);
            }
            if (__any_sync(0xffffffffu, mx[0] > m_[0] + kPaSlack || mx[1] > m_[1] + kPaSlack)) {  // new reference maxima
                float corr[2];
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    mx[h] = fmaxf(mx[h], __shfl_xor_sync(0xffffffffu, mx[h], 4));
                    mx[h] = fmaxf(mx[h], __shfl_xor_sync(0xffffffffu, mx[h], 8));
                    mx[h] = fmaxf(mx[h], __shfl_xor_sync(0xffffffffu, mx[h], 16));
                    const float mnew = fmaxf(m_[h], mx[h]);
                    corr[h] = mnew == -INFINITY ? 1.f : ex2(m_[h] - mnew);
                    m_[h] = mnew;
                    l_[h] *= corr[h];
                }
#pragma unroll
                for (int mt = 0; mt < KS; ++mt) {
                    o[mt][0] *= corr[0]; o[mt][1] *= corr[1];
                    o[mt][2] *= corr[0]; o[mt][3] *= corr[1];
                }
            }
#pragma unroll
            for (int h = 0; h < 2; ++h) mx[h] = m_[h] == -INFINITY ? 0.f : m_[h];  // (nothing seen yet)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                pv[e] = ex2(fmaf(s[e], cm2[e & 1], -mx[e & 1]));
                const int at = pos + (e >> 1) * 8;
                if (!full && (at < t0 || at >= t1)) pv[e] = 0.f;
                l_[e & 1] += pv[e];  // this lane's positions
                pv[e] *= kPaGain;
            }
            uint32_t ph[2], pl[2];
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                __half h0 = __float2half_rn(pv[2 * j]), h1 = __float2half_rn(pv[2 * j + 1]);
                if (HL || PK) {
                    const __half l0 = __float2half_rn(pv[2 * j] - __half2float(h0)), l1 = __float2half_rn(pv[2 * j + 1] - __half2float(h1));
                    if (HL) pl[j] = movm_t(pack_h2(l0, l1));
                    if (PK && c >= 2) { h0 = l0; h1 = l1; }
                }
                ph[j] = movm_t(pack_h2(h0, h1));
            }
#pragma unroll
            for (int mt = 0; mt < KS; ++mt) {
                uint32_t a[4];
                ldsm_x4_t(vs_a + 2 * attn_swz<D>((li >> 1) * 8 + lr, mt * 2 + (li & 1)), a);
                mma16816_acc(o[mt], a[0], a[1], a[2], a[3], ph[0], ph[1]);
                if (HL) mma16816_acc(o[mt], a[0], a[1], a[2], a[3], pl[0], pl[1]);
            }
            __syncwarp();  // the stage is free
            load(b + NST - 1);
        }
        cp_async_wait<0>();
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            float x = l_[h];
            x += __shfl_xor_sync(0xffffffffu, x, 4);
            x += __shfl_xor_sync(0xffffffffu, x, 8);
            x += __shfl_xor_sync(0xffffffffu, x, 16);
            l_[h] = x * kPaGain;
            m_[h] = seen_max(m_[h], x);
        }
    }
    const int ns = p.nss + p.nsp;
    if constexpr (!WHOLE) {
        if (nb > 0) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int col = 2 * c + h;
                const bool mine = col < p.G;  // (PK: the lo columns' outputs are added to the hi columns')
                const size_t at = ((size_t)r * p.heads + kvh * p.G + min(col, p.G - 1)) * ns + p.nss + split;
#pragma unroll
                for (int mt = 0; mt < KS; ++mt)
#pragma unroll
                    for (int k = 0; k < 2; ++k) {
                        float x = o[mt][2 * k + h];
                        if (PK) x += __shfl_xor_sync(0xffffffffu, x, 2);
                        if (mine) p.part_o[at * D + mt * 16 + gq + 8 * k] = x;
                    }
                if (mine && gq == 0) p.part_ml[at] = make_float2(m_[h], l_[h]);
            }
        }
        if (blockIdx.x == 0) pdl_wait();  // this kernel's end then stands for the shared items' too
    } else {
        __shared__ float2 wml[NW][8];
        __syncthreads();  // every warp is done with its ring: it takes the warps' outputs
        float* red = reinterpret_cast<float*>(smem);  // [warp][column][D + 4]
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int col = 2 * c + h;
            const bool mine = col < p.G;
#pragma unroll
            for (int mt = 0; mt < KS; ++mt)
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    float x = o[mt][2 * k + h];
                    if (PK) x += __shfl_xor_sync(0xffffffffu, x, 2);
                    if (mine) red[((size_t)warp * 8 + col) * (D + 4) + mt * 16 + gq + 8 * k] = x;
                }
            if (mine && gq == 0) wml[warp][col] = make_float2(m_[h], l_[h]);
        }
        __syncthreads();
        const int live_s = v.shared > 0 ? (v.shared + p.ls * p.lc - 1) / (p.ls * p.lc) : 0;
        if (live_s || blockIdx.x == 0) pdl_wait();  // the shared items' results
        bool odd = false;
        for (int e = threadIdx.x; e < p.G * (D / 4); e += NW * 32) {
            const int col = e / (D / 4), d = e % (D / 4) * 4, head = kvh * p.G + col;
            const size_t at = ((size_t)r * p.heads + head) * ns;
            float M = -INFINITY, L = 0.f;
            float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
            auto add = [&](float2 ml, const float4& x, float top) {
                if (ml.x == -INFINITY) return;
                const float w = ex2(ml.x - top);
                L = fmaf(ml.y, w, L);
                a.x = fmaf(x.x, w, a.x); a.y = fmaf(x.y, w, a.y);
                a.z = fmaf(x.z, w, a.z); a.w = fmaf(x.w, w, a.w);
            };
#pragma unroll
            for (int w = 0; w < NW; ++w) M = fmaxf(M, wml[w][col].x);
            // the shared items' results, up to four at a time against the maximum so far
#pragma unroll
            for (int w = 0; w < NW; ++w)
                add(wml[w][col], *reinterpret_cast<const float4*>(red + ((size_t)w * 8 + col) * (D + 4) + d), M);
            for (int q0 = 0; q0 < live_s; q0 += 4) {
                float2 ml[4];
                float4 x[4];
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    ml[q] = make_float2(-INFINITY, 0.f);
                    if (q0 + q < live_s) {
                        ml[q] = p.part_ml[at + q0 + q];
                        x[q] = *reinterpret_cast<const float4*>(p.part_o + (at + q0 + q) * D + d);
                    }
                }
                const float top = fmaxf(fmaxf(M, fmaxf(ml[0].x, ml[1].x)), fmaxf(ml[2].x, ml[3].x));
                if (top > M) {
                    const float corr = ex2(M - top);
                    L *= corr;
                    a.x *= corr; a.y *= corr; a.z *= corr; a.w *= corr;
                    M = top;
                }
#pragma unroll
                for (int q = 0; q < 4; ++q) add(ml[q], x[q], M);
            }
            const float iv = M == -INFINITY ? 0.f : 1.f / L;
            T* dst = static_cast<T*>(p.out) + (size_t)r * p.ldo + (size_t)head * D + d;
            const float x[4] = {a.x * iv, a.y * iv, a.z * iv, a.w * iv};
            if (p.out_vec) {
                if constexpr (sizeof(T) == 4) {
                    *reinterpret_cast<float4*>(dst) = make_float4(x[0], x[1], x[2], x[3]);
                } else {
                    const __half2 y = __floats2half2_rn(x[0], x[1]), z = __floats2half2_rn(x[2], x[3]);
                    *reinterpret_cast<uint2*>(dst) = make_uint2(*reinterpret_cast<const uint32_t*>(&y), *reinterpret_cast<const uint32_t*>(&z));
                }
            } else {
#pragma unroll
                for (int k = 0; k < 4; ++k) dst[k] = kv_out<T>(x[k]);
            }
            const float z = (a.x + a.y) + (a.z + a.w);
            odd |= z - z != 0.f && L == L;
        }
        if (odd) {
#pragma unroll 1
            for (int e = threadIdx.x; e < p.G * (D / 4); e += NW * 32) {
                const int d = e % (D / 4) * 4;
                odd_outputs(p, r, kvh, D, d, static_cast<T*>(p.out) + (size_t)r * p.ldo + (size_t)(kvh * p.G + e / (D / 4)) * D + d, 4);
            }
        }
    }
}

// One tile of a group's columns over a split of the shared positions:
// item i of [group][column tile][kv head][split].
template <int D, int NT, typename T>
__device__ __forceinline__ void shared_item(const KvAttnParams& p, int i, int* lim, int* page_ids, float* cmul, int* range,
                                            uint8_t* smem) {
    const int tid = threadIdx.x, split = i % p.nss;
    i /= p.nss;
    const int kvh = i % p.kv_heads;
    i /= p.kv_heads;
    const int ct = i % p.ctiles, g = i / p.ctiles;
    int r0, r1;
    if (!group_rows(p, g, r0, r1)) return;
    const int col0 = ct * NT * 8, ncol = (r1 - r0) * p.G;
    if (col0 >= ncol) return;
    const RowAt lead = row_at(p, r0);
    const int shared = group_shared(p, g);
    if (tid < 32) {
        int n = 0;
        if (tid < NT * 8) {
            const int col = col0 + tid;
            if (col < ncol) n = max(0, row_view(p, r0 + col / p.G, shared).shared);
            lim[tid] = n;
        }
        const int mx = __reduce_max_sync(0xffffffffu, n);
        const int mn = __reduce_min_sync(0xffffffffu, tid < NT * 8 && col0 + tid < ncol ? n : 0x7fffffff);
        if (tid == 0) { range[0] = mx; range[1] = mn; }
    }
    __syncthreads();
    const int t0 = split * p.ls, t1 = min(range[0], t0 + p.ls);
    if (t0 >= t1) return;  // no row of the tile sees this far
    pa_item<D, NT, T>(p, r0, col0, ncol, kvh, group_seq(p, r0, r1, lead), t0, t1, split, lim, range[1], page_ids, cmul, smem);
}

// Grid: the shared items.
template <int D, int NT, typename T>
__global__ void __launch_bounds__(kPaWarps * 32, D == 128 ? 2 : 4) paged_attn_kernel(const KvAttnParams p) {
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ int lim[NT * 8], page_ids[kPaMaxSplit / 16 + 2], range[2];
    __shared__ float cmul[NT * 8];
    pdl_wait();               // what the stream held before this call
    pdl_launch_dependents();  // the private items need nothing of this kernel
    shared_item<D, NT, T>(p, blockIdx.x, lim, page_ids, cmul, range, smem);
}

constexpr int kPmWarps = 4;
// Join the items of a (row, head) pair: a CTA per pair, its warps take every fourth item (one warp alone
// walked a long row's 32 items in 21 us on 64 rows of 32 heads, four take 8), their sums meet in shared
// memory. Latency bounds it: lengths, groups and then the partials, three dependent reads.
template <int D, typename T>
__global__ void __launch_bounds__(kPmWarps * 32) paged_merge_kernel(const KvAttnParams p) {
    constexpr int E = D / 32, U = 8;  // U items' loads in flight
    __shared__ int found;
    __shared__ float acc_s[kPmWarps][D], l_s[kPmWarps], m_s[kPmWarps];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int r = blockIdx.x / p.heads, h = blockIdx.x % p.heads;
    const int len = p.len[r], sq = p.seq ? p.seq[r] : r;
    int shared = 0;
    if (p.groups) {
        if (threadIdx.x == 0) found = 0;
        __syncthreads();
        find_group(p, r, threadIdx.x, kPmWarps * 32, &found);
        __syncthreads();
        shared = found;
    }
    const RowView v = row_view(p, len, sq, shared);
    pdl_wait();
    if (v.n < 0) return;
    const int ns = p.nss + p.nsp;
    const int priv = min(v.n - v.shared, p.max_private);
    if (v.n - v.shared > p.max_private && threadIdx.x == 0) kv_flag(p.err, kKvBadPos);
    const int live_s = v.shared > 0 ? (v.shared + p.ls * p.lc - 1) / (p.ls * p.lc) : 0;
    const int live = live_s + (priv > 0 ? (priv + p.lp - 1) / p.lp : 0);
    const size_t base = (size_t)blockIdx.x * ns;
    auto slot = [&](int i) { return i < live_s ? i : p.nss + (i - live_s); };
    // this warp's items i = warp, warp + 4, ...: U at a time against the running maximum
    float M = -INFINITY, L = 0.f, acc[E] = {};
    for (int i0 = warp; i0 < live; i0 += kPmWarps * U) {
        float2 ml[U];
        float x[U][E];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int i = i0 + u * kPmWarps;
            ml[u] = make_float2(-INFINITY, 0.f);
            if (i < live) {
                ml[u] = p.part_ml[base + slot(i)];
                const float* src = p.part_o + (base + slot(i)) * D + lane * E;
                if constexpr (E == 4) *reinterpret_cast<float4*>(x[u]) = *reinterpret_cast<const float4*>(src);
                else if constexpr (E == 2) *reinterpret_cast<float2*>(x[u]) = *reinterpret_cast<const float2*>(src);
                else x[u][0] = *src;
            }
        }
        float top = M;
#pragma unroll
        for (int u = 0; u < U; ++u) top = fmaxf(top, ml[u].x);
        if (top == -INFINITY) continue;
        const float corr = ex2(M - top);
        M = top;
        L *= corr;
#pragma unroll
        for (int e = 0; e < E; ++e) acc[e] *= corr;
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (ml[u].x != -INFINITY) {
                const float w = ex2(ml[u].x - M);
                L = fmaf(ml[u].y, w, L);
#pragma unroll
                for (int e = 0; e < E; ++e) acc[e] = fmaf(x[u][e], w, acc[e]);
            }
    }
#pragma unroll
    for (int e = 0; e < E; ++e) acc_s[warp][lane * E + e] = acc[e];
    if (lane == 0) { m_s[warp] = M; l_s[warp] = L; }
    __syncthreads();
    float top = -INFINITY, sum = 0.f, w[kPmWarps];
#pragma unroll
    for (int k = 0; k < kPmWarps; ++k) top = fmaxf(top, m_s[k]);
#pragma unroll
    for (int k = 0; k < kPmWarps; ++k) {
        w[k] = m_s[k] == -INFINITY ? 0.f : ex2(m_s[k] - top);
        sum = fmaf(l_s[k], w[k], sum);
    }
    const float iv = top == -INFINITY ? 0.f : 1.f / sum;
    T* dst = static_cast<T*>(p.out) + (size_t)r * p.ldo + (size_t)h * D;
    for (int d = threadIdx.x; d < D; d += kPmWarps * 32) {
        float a = 0.f;
#pragma unroll
        for (int k = 0; k < kPmWarps; ++k)
            if (m_s[k] != -INFINITY) a = fmaf(acc_s[k][d], w[k], a);
        dst[d] = kv_out<T>(a * iv);
        if (a - a != 0.f && sum == sum) odd_outputs(p, r, h / p.G, D, d, dst + d, 1);
    }
}

}  // namespace laic
