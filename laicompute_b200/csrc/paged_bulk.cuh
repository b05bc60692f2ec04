// The bulk of a shared prefix on the 5th-generation tensor cores.
//
// A group with many columns (rows x query heads of one KV head) makes its attention a pair of dense
// products: S = Q K^T and O += P V over 256 columns per CTA, two tiles of M = 128. Only positions
// that every column of the CTA sees come here, in whole tiles of kBulkKeys, so no mask enters; the
// rest of each column's positions is left to the items of paged_attn.cuh, and the merge joins all.
//
// Roles: warp 8 loads (one lane: TMA boxes of up to a page, 128-byte swizzle, a ring of K + V
// stages); warp 9 multiplies (one lane: tcgen05.mma, S and O in tensor memory, P read from tensor
// memory, where it takes S's place); warps 0-3 and 4-7 each own a tile, a thread a column: they read
// S, keep the running maximum and sum, and write P. The issue order PV(j), QK(j + 1) per tile lets
// one tile's products run under the other's exponentials. O is rescaled only when a maximum grew by
// more than 2^8 since the last time (weights stay below 2^15 in binary16 with the factor 2^7 they
// carry); both tiles' accumulators fill the 512 columns of tensor memory.
//
// FP32 rows: Q as binary16 hi + lo after a scaling by a power of two, P likewise, the lo products
// first (the accumulators then start from small terms), 64 keys per tile; binary16 rows: one product
// each, P rounded to binary16, 128 keys per tile.
#pragma once
#include <cuda.h>

#include "paged_attn.cuh"

namespace laic {

constexpr int kBulkThreads = 320;
constexpr int kBulkMaxSplit = 2048;   // positions per item at most (its page ids are in shared memory)
constexpr float kBulkSlack = 8.f;     // log2 of how far a maximum may outgrow its reference

__host__ __device__ constexpr int bulk_keys(bool f32) { return f32 ? 64 : 128; }
__host__ __device__ constexpr int bulk_stage_bytes(int D, bool f32) { return 2 * bulk_keys(f32) * D * 2; }
__host__ __device__ constexpr int bulk_q_bytes(int D, bool f32) { return kBulkCols * D * 2 * (f32 ? 2 : 1); }
__host__ __device__ constexpr int bulk_stages(int D, bool f32) { return D == 64 ? 4 : f32 ? 3 : 2; }
__host__ __device__ constexpr int bulk_smem(int D, bool f32) {
    return bulk_q_bytes(D, f32) + bulk_stages(D, f32) * bulk_stage_bytes(D, f32) + 1024;  // (aligned to 1024)
}

// ---- PTX
__device__ __forceinline__ void tma_2d(uint32_t dst, const CUtensorMap* map, int x, int y, uint64_t* bar) {
    asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];"
                 ::"r"(dst), "l"(map), "r"(x), "r"(y), "r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void tc_alloc(uint32_t smem_dst, uint32_t cols) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_dst), "r"(cols) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
}
__device__ __forceinline__ void tc_dealloc(uint32_t addr, uint32_t cols) {
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(addr), "r"(cols));
}
__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_commit(uint64_t* bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}
// D (tensor memory) (+)= A B, A and B in shared memory / A in tensor memory
__device__ __forceinline__ void tc_mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool acc) {
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %4, 0;\n\t"
                 "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}"
                 ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"((uint32_t)acc) : "memory");
}
__device__ __forceinline__ void tc_mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, bool acc) {
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %4, 0;\n\t"
                 "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
                 ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"((uint32_t)acc) : "memory");
}
__device__ __forceinline__ void tc_ld32(uint32_t addr, uint32_t* r) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
        "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
          "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
          "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(addr));
}
__device__ __forceinline__ void tc_st32(uint32_t addr, const uint32_t* r) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
        "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};"
        ::"r"(addr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]),
        "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]),
        "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]),
        "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
        : "memory");
}
__device__ __forceinline__ void tc_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
// The values of a tc_ld32 once tc_wait_ld has returned: uses of them cannot move above this.
__device__ __forceinline__ void tc_loaded(uint32_t* r) {
    asm volatile("" : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]),
                       "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]), "+r"(r[16]), "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]), "+r"(r[22]), "+r"(r[23]),
                       "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]), "+r"(r[29]), "+r"(r[30]), "+r"(r[31]));
}
__device__ __forceinline__ void tc_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// Shared-memory operand descriptor, 128-byte swizzle: start, strides between core groups (bytes).
__device__ __forceinline__ uint64_t umma_desc(uint32_t addr, uint32_t lbo, uint32_t sbo) {
    return (uint64_t)((addr & 0x3ffff) >> 4) | (uint64_t)(lbo >> 4) << 16 | (uint64_t)(sbo >> 4) << 32 | (uint64_t)1 << 46 |
           (uint64_t)2 << 61;
}
// kind::f16, binary16 operands, FP32 accumulator, M = 128; bmn: B's N dimension is the contiguous one.
__host__ __device__ constexpr uint32_t umma_idesc(int n, bool bmn) {
    return 1u << 4 | (bmn ? 1u << 16 : 0u) | (uint32_t)(n >> 3) << 17 | (uint32_t)(128 >> 4) << 24;
}

// A bounded wait (about a second of SM clocks) for a barrier phase. Once one of the CTA's waits has
// run out (*dead), the others stop at once.
__device__ __forceinline__ bool bulk_wait(uint64_t* bar, uint32_t parity, volatile int* dead, int* err) {
    if (mbar_try_wait(bar, parity)) return true;
    const long long t0 = clock64();
    while (!mbar_try_wait_sleep(bar, parity)) {
        if (*dead) return false;
        if (clock64() - t0 > 2000000000LL) {
            *dead = 1;
            kv_flag(err, kKvWait);
            return false;
        }
    }
    return true;
}

// Grid [group][pair][kv head][split].
template <int D, typename T>
__global__ void __launch_bounds__(kBulkThreads, 1) paged_bulk_kernel(const KvAttnParams p, const __grid_constant__ CUtensorMap mk,
                                                                     const __grid_constant__ CUtensorMap mv) {
    constexpr bool F32 = sizeof(T) == 4;
    constexpr int HN = F32 ? 2 : 1, NK = bulk_keys(F32), NS = bulk_stages(D, F32), HALVES = D / 64;
    constexpr int STAGE = bulk_stage_bytes(D, F32), VOFF = STAGE / 2;
    constexpr int QPART = 128 * D * 2;  // one tile's hi or lo part
    extern __shared__ uint8_t dyn[];
    uint8_t* base = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(dyn) + 1023) & ~(uintptr_t)1023);
    uint8_t* stages = base + bulk_q_bytes(D, F32);
    __shared__ int page_ids[kBulkMaxSplit / 16 + 2];
    __shared__ uint64_t kv_full[NS], kv_free[NS], s_full[2], p_ready[2], o_done;
    __shared__ uint32_t tmem_at;
    __shared__ volatile int dead;
    __shared__ int s_bulk;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;

    int i = blockIdx.x;
    const int split = i % p.nbs;
    i /= p.nbs;
    const int kvh = i % p.kv_heads;
    i /= p.kv_heads;
    const int pair = i % p.pairs, g = i / p.pairs;
    int r0, r1;
    if (!group_rows(p, g, r0, r1)) return;
    const int ncol = (r1 - r0) * p.G, col0 = pair * kBulkCols;
    if (col0 >= ncol) return;
    if (warp == 0) {
        const int n = pair_bulk(p, r0, r1, pair, group_shared(p, g, r0), lane);
        if (lane == 0) s_bulk = n;
    }
    if (tid == 0) dead = 0;
    __syncthreads();
    const int t0 = split * p.lb, t1 = min(s_bulk, t0 + p.lb);
    if (t0 >= t1) return;
    const int seq = row_seq(p, r0);
    const int nt = (t1 - t0) / NK;
    const int tiles = ncol - col0 > 128 ? 2 : 1;  // M tiles with columns

    // ---- set-up: page ids, barriers, tensor memory, Q
    const int first_page = t0 >> p.page_shift, npages = ((t1 - 1) >> p.page_shift) - first_page + 1;
    for (int k = tid; k < npages; k += kBulkThreads) {
        int id = p.table[(size_t)seq * p.pages_per_seq + first_page + k];
        if (id < 0 || id >= p.num_pages) {
            kv_flag(p.err, kKvBadPage);
            id = 0;
        }
        page_ids[k] = id;
    }
    if (tid == 0) {
        for (int s = 0; s < NS; ++s) { mbar_init(&kv_full[s], 1); mbar_init(&kv_free[s], 1); }
        for (int w = 0; w < 2; ++w) { mbar_init(&s_full[w], 1); mbar_init(&p_ready[w], 128); }
        mbar_init(&o_done, 1);
        mbar_fence_init();
    }
    if (warp == 9) tc_alloc(smem_u32(&tmem_at), 512);
    const int wg = warp >> 2, row = tid & 127, col = col0 + tid;  // a softmax thread's column (tid < 256)
    const bool live = tid < 256 && col < ncol;
    const int rr = r0 + (live ? col / p.G : 0), hh = kvh * p.G + (live ? col % p.G : 0);
    float cm = 0.f;
    if (tid < 256 && wg < tiles) {
        const T* q = static_cast<const T*>(p.q) + (size_t)rr * p.ldq + (size_t)hh * D;
        uint8_t* qs = base + (size_t)wg * HN * QPART;
        const float sgn = p.scale_log2 < 0.f ? -1.f : 1.f;  // (the maximum is taken of S itself)
        float fac = sgn, inv = 1.f;
        if constexpr (F32) {
            float mx = 0.f;
            for (int d = 0; live && d < D; d += 4) {
                float4 x;
                if (p.q_vec) x = *reinterpret_cast<const float4*>(q + d);
                else x = make_float4(q[d], q[d + 1], q[d + 2], q[d + 3]);
                mx = fmaxf(fmaxf(mx, fmaxf(fabsf(x.x), fabsf(x.y))), fmaxf(fabsf(x.z), fabsf(x.w)));
            }
            const int e = min(max((int)(__float_as_uint(mx) >> 23) - 127, -100), 120);
            fac = sgn * __uint_as_float((uint32_t)(127 - e) << 23);
            inv = __uint_as_float((uint32_t)(127 + e) << 23);
        }
        cm = fabsf(p.scale_log2) * inv;
#pragma unroll
        for (int ch = 0; ch < D / 8; ++ch) {  // 16-byte chunks of the row
            float x[8];
            if (live) {
                if (p.q_vec) {
                    Raw8<T> raw;
                    load8<T, true>(q + ch * 8, raw);
#pragma unroll
                    for (int k = 0; k < 8; ++k) x[k] = raw.at(k) * fac;
                } else {
#pragma unroll
                    for (int k = 0; k < 8; ++k) x[k] = kv_in<T>(q[ch * 8 + k]) * fac;
                }
            } else {
#pragma unroll
                for (int k = 0; k < 8; ++k) x[k] = 0.f;
            }
            uint32_t hi[4], lo[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const __half a = __float2half_rn(x[2 * k]), b = __float2half_rn(x[2 * k + 1]);
                hi[k] = pack_h2(a, b);
                lo[k] = pack_h2(__float2half_rn(x[2 * k] - __half2float(a)), __float2half_rn(x[2 * k + 1] - __half2float(b)));
            }
            const int at = (ch >> 3) * (128 * 128) + row * 128 + (((ch & 7) ^ (row & 7)) << 4);
            *reinterpret_cast<uint4*>(qs + at) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
            if constexpr (F32) *reinterpret_cast<uint4*>(qs + QPART + at) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    pdl_launch_dependents();  // the items kernel needs nothing of this one
    const uint32_t tmem = tmem_at;
    auto s_at = [&](int w) { return tmem + (uint32_t)(w * NK); };        // S, then P hi | P lo in its place
    auto o_at = [&](int w) { return tmem + 256u + (uint32_t)(w * D); };

    if (warp == 8) {
        if (lane == 0) {
            const int box = min(1 << p.page_shift, NK);  // rows of a TMA box
            int j = 0;
            for (; j < nt; ++j) {
                const int s = j % NS;
                if (j >= NS && !bulk_wait(&kv_free[s], (uint32_t)(j / NS - 1) & 1, &dead, p.err)) break;
                mbar_expect_tx(&kv_full[s], STAGE);
                const uint32_t ks = smem_u32(stages) + (uint32_t)(s * STAGE);
                for (int k = 0; k < NK; k += box) {
                    const int t = t0 + j * NK + k;
                    const int y = ((page_ids[(t >> p.page_shift) - first_page] * p.kv_heads + kvh) << p.page_shift) +
                                  (t & ((1 << p.page_shift) - 1));
#pragma unroll
                    for (int h = 0; h < HALVES; ++h) {
                        tma_2d(ks + h * (NK * 128) + k * 128, &mk, h * 64, y, &kv_full[s]);
                        tma_2d(ks + VOFF + h * (NK * 128) + k * 128, &mv, h * 64, y, &kv_full[s]);
                    }
                }
            }
            if (dead)  // copies still in flight land before the CTA's memory is given up
                for (int k = max(0, j - NS); k < j; ++k) {
                    const long long since = clock64();
                    while (!mbar_try_wait(&kv_full[k % NS], (uint32_t)(k / NS) & 1) && clock64() - since < 200000000LL) {}
                }
        }
    } else if (warp == 9) {
        if (lane == 0) {
            constexpr uint32_t iqk = umma_idesc(NK, false), ipv = umma_idesc(D, true);
            bool ok = true;
            auto qk = [&](int w, int j) {
                const uint32_t ks = smem_u32(stages) + (uint32_t)(j % NS * STAGE);
                const uint32_t qa = smem_u32(base) + (uint32_t)(w * HN * QPART);
#pragma unroll
                for (int part = HN - 1; part >= 0; --part)  // lo, then hi
#pragma unroll
                    for (int k = 0; k < D / 16; ++k) {
                        const uint32_t off = (uint32_t)(k & 3) * 32;
                        tc_mma_ss(s_at(w), umma_desc(qa + part * QPART + (k >> 2) * (128 * 128) + off, 16, 1024),
                                  umma_desc(ks + (k >> 2) * (NK * 128) + off, 16, 1024), iqk, part != HN - 1 || k > 0);
                    }
                tc_commit(&s_full[w]);
            };
            auto pv = [&](int w, int j) {
                const uint32_t vs = smem_u32(stages) + (uint32_t)(j % NS * STAGE) + VOFF;
#pragma unroll
                for (int part = HN - 1; part >= 0; --part)
#pragma unroll
                    for (int k = 0; k < NK / 16; ++k)
                        tc_mma_ts(o_at(w), s_at(w) + part * (NK / 2) + k * 8, umma_desc(vs + k * 2048, NK * 128, 1024), ipv,
                                  j > 0 || part != HN - 1 || k > 0);
            };
            ok = bulk_wait(&kv_full[0], 0, &dead, p.err);
            if (ok) {
                tc_fence_after();
                for (int w = 0; w < tiles; ++w) qk(w, 0);
            }
            for (int j = 0; j < nt && ok; ++j)
                for (int w = 0; w < tiles && ok; ++w) {
                    if (!(ok = bulk_wait(&p_ready[w], (uint32_t)j & 1, &dead, p.err))) break;
                    tc_fence_after();
                    pv(w, j);
                    if (w == tiles - 1) tc_commit(&kv_free[j % NS]);
                    if (j + 1 < nt) {
                        if (w == 0 && !(ok = bulk_wait(&kv_full[(j + 1) % NS], (uint32_t)((j + 1) / NS) & 1, &dead, p.err))) break;
                        tc_fence_after();
                        qk(w, j + 1);
                    }
                }
            tc_commit(&o_done);  // after a failed wait too: whatever was issued ends before tensor memory is freed
        }
    } else if (wg < tiles) {
        const uint32_t lane_at = (uint32_t)(warp & 3) * 32u << 16;
        const uint32_t S = s_at(wg) + lane_at, O = o_at(wg) + lane_at;
        float mref = 0.f, l = 0.f;
        bool ok = true;
        for (int j = 0; j < nt; ++j) {
            ok = __all_sync(0xffffffffu, bulk_wait(&s_full[wg], (uint32_t)j & 1, &dead, p.err));
            if (!ok) break;
            tc_fence_after();
            uint32_t s[NK];
#pragma unroll
            for (int k = 0; k < NK; k += 32) tc_ld32(S + k, s + k);
            tc_wait_ld();
#pragma unroll
            for (int k = 0; k < NK; k += 32) tc_loaded(s + k);
            float mx = __uint_as_float(s[0]);
#pragma unroll
            for (int k = 1; k < NK; ++k) mx = fmaxf(mx, __uint_as_float(s[k]));
            mx *= cm;
            if (j == 0) {
                mref = mx == -INFINITY ? 0.f : mx;
            } else if (__any_sync(0xffffffffu, mx > mref + kBulkSlack)) {
                const float next = fmaxf(mref, mx), corr = ex2(mref - next);
                mref = next;
                l *= corr;
#pragma unroll 1
                for (int k = 0; k < D; k += 32) {
                    uint32_t o[32];
                    tc_ld32(O + k, o);
                    tc_wait_ld();
                    tc_loaded(o);
#pragma unroll
                    for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * corr);
                    tc_st32(O + k, o);
                }
            }
            float sum0 = 0.f, sum1 = 0.f;
#pragma unroll
            for (int k = 0; k < NK; k += 64) {  // 64 positions: 32 words of hi, 32 of lo
                uint32_t hi[32], lo[F32 ? 32 : 1];
#pragma unroll
                for (int e = 0; e < 32; ++e) {
                    float a = ex2(fmaf(__uint_as_float(s[k + 2 * e]), cm, -mref));
                    float b = ex2(fmaf(__uint_as_float(s[k + 2 * e + 1]), cm, -mref));
                    sum0 += a;
                    sum1 += b;
                    a *= kPaGain;
                    b *= kPaGain;
                    const __half2 h = __floats2half2_rn(a, b);
                    hi[e] = *reinterpret_cast<const uint32_t*>(&h);
                    if constexpr (F32) {
                        const float2 f = __half22float2(h);
                        const __half2 r = __floats2half2_rn(a - f.x, b - f.y);
                        lo[e] = *reinterpret_cast<const uint32_t*>(&r);
                    }
                }
                tc_st32(S + k / 2, hi);
                if constexpr (F32) tc_st32(S + NK / 2 + k / 2, lo);
            }
            l += sum0 + sum1;
            tc_wait_st();
            tc_fence_before();
            mbar_arrive(&p_ready[wg]);
        }
        ok = __all_sync(0xffffffffu, bulk_wait(&o_done, 0, &dead, p.err)) && ok;
        tc_fence_after();
        if (ok) {
            const int ns = p.nbs + p.nss + p.nsp;
            const size_t at = ((size_t)rr * p.heads + hh) * ns + split;
#pragma unroll 1
            for (int k = 0; k < D; k += 32) {
                uint32_t o[32];
                tc_ld32(O + k, o);
                tc_wait_ld();
                tc_loaded(o);
                if (live) {
                    uint4* dst = reinterpret_cast<uint4*>(p.part_o + at * D + k);
#pragma unroll
                    for (int e = 0; e < 8; ++e) dst[e] = make_uint4(o[4 * e], o[4 * e + 1], o[4 * e + 2], o[4 * e + 3]);
                }
            }
            if (live) p.part_ml[at] = make_float2(mref, l * kPaGain);
        }
        tc_fence_before();
    }
    __syncwarp();
    __syncthreads();
    if (warp == 9) {
        if (lane == 0) bulk_wait(&o_done, 0, &dead, p.err);
        __syncwarp();
        tc_fence_after();
        tc_dealloc(tmem, 512);
    }
}

}  // namespace laic
