// Shared positions of wide groups on the 5th-generation tensor cores.
//
// A group with many columns (rows x query heads of one KV head) makes its attention a pair of dense
// products: S = Q K^T and O += P V over one or two tiles of M = 128 columns per CTA (two from 129 columns
// on: one tile's softmax then runs under the other's products) and a split of the group's positions, 128
// at a time.
//
// Roles: a warpgroup per tile, a thread a column: it reads S, keeps the running maximum and sum, and
// writes P in two halves, so that PV starts on the first; a warp that loads (TMA boxes of up to a page,
// 128-byte swizzle, a lane per box: one lane alone took 125 cycles a box, 4,000 for a tile of 16-position
// pages; a ring of K and V tiles; its first loads start while the others bring Q); two warps that
// multiply (one lane each: tcgen05.mma, S and O in tensor memory, P read from tensor memory, where
// it takes S's place).
// Binary16 rows, where a tile's exponentials take longer than its products: one lane multiplies for
// both tiles in turn, which keeps one tile's products under the other's exponentials (512 prompt rows
// behind 1,537 positions, 32 heads over 8 of 128: 37.3 us; a lane per tile lets them fall into step, 39.3).
// FP32 rows, with twice the products: a lane per tile, which won while a tile's way was longer; now the two are
// alike (64 rows behind 4,101 shared positions: 41.0 us against 41.1; the prompt rows above: 52.1 against 50.1).
// 128 positions per tile: a product of N = 64 takes about as long as one of N = 128 (100 against 85
// cycles), and two score buffers of 64 ran slower than one of 128. O is rescaled only when a maximum
// grew by more than 2^8 since the last time (weights stay below 2^15 in binary16 with the factor 2^7
// they carry). Both tiles' S and O fill the 512 columns of tensor memory. What bounds it: the chain
// softmax -> PV -> QK of a tile (4,200 cycles a pair of 128-position tiles in binary16, of which
// the exponentials fill 2,048 at 16 a clock and the 32 products 2,700; 3,200 for one tile alone), and, for few tiles per CTA,
// the way to the first scores (7,000 to 11,000 cycles: Q for every CTA out of L2) and the join (8,000
// over a cluster's shared memory at about 14 bytes a clock). The prompt rows above run at 404 TFLOP/s; the 64 FP32
// rows over 4,101 shared positions take 16 to 22 us here, of the call's 41.
//
// The splits of a set of columns form a thread-block cluster and join through distributed shared
// memory: one partial per cluster goes to global memory, or the output itself where the cluster holds
// all that its rows see.
//
// Tiles that some column does not see to their end are masked. There 0 * V must not be 0 * inf: the
// softmax threads clear what is not finite in V before the product (all of it past the positions any
// column sees), note the positions, and the columns that do see one take its infinities and NaN at
// the end. An output that is NaN all the same is looked up (odd_output).
//
// FP32 rows: Q as binary16 hi + lo after a scaling by a power of two, P likewise, the lo products
// first (the accumulators then start from small terms); binary16 rows: one product each, P rounded to
// binary16.
#pragma once
#include <cuda.h>

#include <type_traits>

#include "paged_attn.cuh"

namespace laic {

// TILES (1 or 2): M tiles of a CTA
constexpr int kBulkTiles = 2;
constexpr int kBulkThreads = 352;     // with two; a warpgroup per tile, then loads, then two that multiply
__host__ __device__ constexpr int bulk_cols(int tiles) { return 128 * tiles; }  // score columns of a CTA
__host__ __device__ constexpr int bulk_threads(int tiles) { return 128 * tiles + 96; }
constexpr int kBulkMaxCluster = 8;   // clusters of 1, 2, 4 or 8
constexpr int kBulkMaxSplit = 2048;   // positions per item at most (its page ids are in shared memory)

constexpr int kBulkKeys = 128;        // positions per tile
constexpr float kBulkLowest = -3e38f; // the reference of a column that has seen no finite score
constexpr int kBulkEarly = 2;         // ring items loaded before the CTA meets (a box takes 70 to 150 cycles to issue)
__host__ __device__ constexpr int bulk_slot_bytes(int D) { return kBulkKeys * D * 2; }  // a tile of K or of V
__host__ __device__ constexpr int bulk_q_bytes(int D, bool f32, int tiles) { return bulk_cols(tiles) * D * 2 * (f32 ? 2 : 1); }
// (one tile: room for private items' CTAs on the SM)
__host__ __device__ constexpr int bulk_slots(int D, bool f32, int tiles) { return D == 64 ? 6 : f32 ? 3 : tiles == 2 ? 5 : 4; }
__host__ __device__ constexpr int bulk_smem(int D, bool f32, int tiles) {
    return bulk_q_bytes(D, f32, tiles) + bulk_slots(D, f32, tiles) * bulk_slot_bytes(D) + 1024;  // (aligned to 1024)
}
// (at the end the ring and Q hold O's rows and their maxima and sums)
__host__ __device__ constexpr int bulk_rows_bytes(int D, int tiles) { return bulk_cols(tiles) * (D + 4) * 4; }
__host__ __device__ constexpr bool bulk_rows_fit(int D, int tiles) {
    return bulk_smem(D, false, tiles) - 1024 >= bulk_rows_bytes(D, tiles) + bulk_cols(tiles) * 8;
}
static_assert(bulk_rows_fit(64, 1) && bulk_rows_fit(64, 2) && bulk_rows_fit(128, 1) && bulk_rows_fit(128, 2), "O's rows fit");

// ---- PTX
__device__ __forceinline__ void tma_2d(uint32_t dst, const CUtensorMap* map, int x, int y, uint64_t* bar) {
    asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];"
                 ::"r"(dst), "l"(map), "r"(x), "r"(y), "r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void tma_prefetch(const CUtensorMap* map) { asm volatile("prefetch.tensormap [%0];" ::"l"(map) : "memory"); }
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
// 16 columns, waited for
__device__ __forceinline__ void tc_ld16(uint32_t addr, uint32_t* r) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];\n\t"
                 "tcgen05.wait::ld.sync.aligned;"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
                    "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
                 : "r"(addr)
                 : "memory");
}
__device__ __forceinline__ void tc_st16(uint32_t addr, const uint32_t* r) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};"
                 ::"r"(addr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
                  "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
                 : "memory");
}
__device__ __forceinline__ void tc_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
// The values of a tc_ld32 once tc_wait_ld has returned: uses of them cannot move above this.
__device__ __forceinline__ void tc_loaded(uint32_t* r) {
    asm volatile("" : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]),
                       "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]), "+r"(r[16]), "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]), "+r"(r[22]), "+r"(r[23]),
                       "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]), "+r"(r[29]), "+r"(r[30]), "+r"(r[31]));
}
__device__ __forceinline__ float max3(float a, float b, float c) {
    float r;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
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

// Packed pairs of FP32 operations.
__device__ __forceinline__ uint64_t f2_pack(float a, float b) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ void f2_unpack(uint64_t v, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v)); }
__device__ __forceinline__ uint64_t f2_fma(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ uint64_t f2_add(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ uint64_t f2_mul(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}

// Where the clusters write the output themselves, the first CTA leaves the zeros of the rows of no group.
template <int D, typename T>
__device__ __forceinline__ void groupless_rows(const KvAttnParams& p) {
    if (!p.direct || blockIdx.x != 0) return;
    const int lane = threadIdx.x & 31;
    const int g0 = max(0, min(p.rows, p.group_rows[0])), g1 = max(g0, min(p.rows, p.group_rows[p.groups]));
    for (int r = threadIdx.x >> 5; r < p.rows; r += blockDim.x / 32) {
        if (r >= g0 && r < g1) continue;
        const RowView v = row_view(p, r, 0);
        if (v.n < 0) continue;
        if (v.n > 0 && lane == 0) kv_flag(p.err, kKvBadPos);
        for (int e = lane; e < p.heads * D; e += 32) static_cast<T*>(p.out)[(size_t)r * p.ldo + e] = kv_out<T>(0.f);
    }
}

// Grid [group][pair of column tiles][kv head][split], clusters of bulk_cluster consecutive splits.
template <int D, typename T, int TILES>
__global__ void __launch_bounds__(kBulkThreads, 1) paged_bulk_kernel(const KvAttnParams p, const __grid_constant__ CUtensorMap mk,
                                                                     const __grid_constant__ CUtensorMap mv) {
    constexpr bool F32 = sizeof(T) == 4;
    constexpr int HN = F32 ? 2 : 1, NK = kBulkKeys, NS = bulk_slots(D, F32, TILES), HALVES = D / 64;
    constexpr int SLOT = bulk_slot_bytes(D), COLS = bulk_cols(TILES), LOADER = 4 * TILES, MMA = LOADER + 1;  // (warps)
    constexpr int QPART = 128 * D * 2;  // one tile's hi or lo part
    extern __shared__ uint8_t dyn[];
    uint8_t* base = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(dyn) + 1023) & ~(uintptr_t)1023);
    uint8_t* ring = base + bulk_q_bytes(D, F32, TILES);
    __shared__ int page_ids[kBulkMaxSplit / 16 + 2];
    __shared__ uint64_t kv_full[NS], kv_free[NS], s_full[2], p_ready[2][2], pv_half[2], o_done;
    __shared__ uint32_t tmem_at;
    __shared__ volatile int dead;
    __shared__ int lim_max, lim_min;
    __shared__ float cmul[COLS];
    __shared__ uint32_t odd[kBulkMaxSplit / 32];  // positions of the split whose V was not finite in a masked tile
    __shared__ int any_odd;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;

    namespace cg = cooperative_groups;
    cg::cluster_group cluster = cg::this_cluster();
    const int C = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
    if (tid == 0) { tma_prefetch(&mk); tma_prefetch(&mv); }
    pdl_wait();  // what the stream held before this call
    int i = blockIdx.x;
    const int nsplit = p.nss * C, split = i % nsplit;
    i /= nsplit;
    const int kvh = i % p.kv_heads;
    i /= p.kv_heads;
    const int pair = i % p.ctiles, g = i / p.ctiles;
    int r0, r1;
    const int glen = p.group_len[g];
    if (!group_rows(p, g, r0, r1)) r1 = r0;
    const int ncol = (r1 - r0) * p.G, col0 = pair * COLS;
    if (col0 >= ncol) {  // (alike for all CTAs of a cluster)
        groupless_rows<D, T>(p);
        return;
    }
    const int t0 = split * p.ls;
    const int shared = max(0, kv_clamp_len(p, glen, p.max_shared));
    const int tiles = TILES == 2 && ncol - col0 > 128 ? 2 : 1;  // M tiles with columns

    // ---- a softmax thread's column and how far it sees
    const int wg = warp >> 2, col = col0 + tid;
    const bool live = tid < COLS && col < ncol;
    const int base_row = col0 / p.G, base_head = col0 - base_row * p.G;  // of the pair's first column
    // column cw of the pair: its row and query head (cw + base_head < 2^9: the product by 2^16 / G rounds right)
    auto row_of = [&](int cw) { return (int)((uint32_t)(cw + base_head) * p.g_inv >> 16); };
    const int my_row = row_of(live ? tid : 0);
    const int rr = r0 + base_row + my_row;
    const int my_len = p.len[rr], my_seq = p.seq ? p.seq[rr] : rr;  // under way while Q is loaded
    const int first_page = t0 >> p.page_shift;

    // ring item m: K of tile m / 2, then its V; a lane per box: (piece of the tile, half of the row)
    auto slot = [&](int m) { return smem_u32(ring) + (uint32_t)(m % NS * SLOT); };
    auto load = [&](int m, int t1) {
        const int box = min(1 << p.page_shift, NK), half = lane % HALVES, k = lane / HALVES * box, s = m % NS;
        if (lane == 0) mbar_expect_tx(&kv_full[s], SLOT);
        __syncwarp();
        if (lane < NK / box * HALVES) {
            const int t = t0 + (m >> 1) * NK + k;
            int id = 0;  // past the last position seen: any page (masked, and cleared in V)
            if (t < t1) {
                id = page_ids[(t >> p.page_shift) - first_page];
                if (id < 0 || id >= p.num_pages) {
                    kv_flag(p.err, kKvBadPage);
                    id = 0;
                }
            }
            const int y = ((id * p.kv_heads + kvh) << p.page_shift) + (t & ((1 << p.page_shift) - 1));
            tma_2d(slot(m) + half * (NK * 128) + k * 128, m & 1 ? &mv : &mk, half * 64, y, &kv_full[s]);
        }
    };
    if (warp == LOADER) {  // the first loads, while the others bring Q: the chain lengths -> sequence -> pages is its own
        if (lane == 0) {
            for (int s = 0; s < NS; ++s) { mbar_init(&kv_full[s], 1); mbar_init(&kv_free[s], F32 ? tiles : 1); }
            for (int w = 0; w < 2; ++w) {
                mbar_init(&s_full[w], 1);
                mbar_init(&pv_half[w], 1);
                for (int h = 0; h < 2; ++h) mbar_init(&p_ready[w][h], 128);
            }
            mbar_init(&o_done, F32 ? tiles : 1);
            mbar_fence_init();
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        }
        const RowAt lead = row_at(p, r0);
        // (rows that see nothing do not keep the others' tiles from being whole)
        int hi = 0, lo = 0x7fffffff;
        for (int k = lane; k <= row_of(min(COLS, ncol - col0) - 1); k += 32) {
            const int n = row_view(p, r0 + base_row + k, shared).shared;
            if (n > 0) { hi = max(hi, n); lo = min(lo, n); }
        }
        hi = __reduce_max_sync(0xffffffffu, hi);
        lo = __reduce_min_sync(0xffffffffu, lo);
        const int seq = group_seq(p, r0, r1, lead);
        const int npages = min(((t0 + p.ls - 1) >> p.page_shift) + 1, p.pages_per_seq) - first_page;
        for (int k = lane; k < npages; k += 32) page_ids[k] = p.table[(size_t)seq * p.pages_per_seq + first_page + k];
        if (lane == 0) { lim_max = hi; lim_min = lo; }
        __syncwarp();
        const int t1 = min(hi, t0 + p.ls), items = t0 < t1 ? 2 * ((t1 - t0 + NK - 1) / NK) : 0;
        for (int m = 0; m < min(kBulkEarly, items); ++m) load(m, t1);
    }
    if (warp == MMA) tc_alloc(smem_u32(&tmem_at), 256 * TILES);

    // ---- Q in 128-byte swizzled rows
    auto q_at = [&](int cw) {  // row of q of the pair's column cw
        const int qr = row_of(cw);
        return static_cast<const T*>(p.q) + (size_t)(r0 + base_row + qr) * p.ldq + (size_t)(kvh * p.G + cw + base_head - qr * p.G) * D;
    };
    auto q_dst = [&](int cw, int ch) {  // 16-byte chunk ch of its binary16 row
        const int row = cw & 127;
        return base + (size_t)(cw >> 7) * HN * QPART + (ch >> 3) * (128 * 128) + row * 128 + (((ch & 7) ^ (row & 7)) << 4);
    };
    constexpr int CH = D / 8;  // chunks per row
    if (warp >= LOADER) {
    } else if constexpr (!F32) {
        for (int k = tid; k < tiles * 128 * CH; k += COLS) {
            const int cw = k / CH, ch = k % CH;
            const bool in = col0 + cw < ncol;
            if (p.q_vec) {
                cp_async16_z(smem_u32(q_dst(cw, ch)), in ? q_at(cw) + ch * 8 : static_cast<const T*>(p.q), in);
            } else {
                __half x[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) x[e] = in ? q_at(cw)[ch * 8 + e] : __float2half_rn(0.f);
                *reinterpret_cast<uint4*>(q_dst(cw, ch)) = *reinterpret_cast<const uint4*>(x);
            }
        }
        cmul[tid] = p.scale_log2;
        cp_async_commit();
        cp_async_wait_all();
    } else if (warp < 4 * tiles) {
        // a warp takes 32 columns, CH lanes a row; eight steps' loads in flight
        constexpr int RPI = 32 / CH, STEPS = 32 / RPI, B = 8;
        const int sub = lane / CH, ch = lane % CH;
#pragma unroll 1
        for (int it0 = 0; it0 < STEPS; it0 += B) {
            float xs[B][8];
#pragma unroll
            for (int b = 0; b < B; ++b) {
                const int cw = warp * 32 + (it0 + b) * RPI + sub;
                float* x = xs[b];
#pragma unroll
                for (int e = 0; e < 8; ++e) x[e] = 0.f;
                if (col0 + cw < ncol) {
                    const float* q = reinterpret_cast<const float*>(q_at(cw)) + ch * 8;
                    if (p.q_vec) {
                        *reinterpret_cast<float4*>(x) = *reinterpret_cast<const float4*>(q);
                        *reinterpret_cast<float4*>(x + 4) = *reinterpret_cast<const float4*>(q + 4);
                    } else {
#pragma unroll
                        for (int e = 0; e < 8; ++e) x[e] = q[e];
                    }
                }
            }
#pragma unroll
            for (int b = 0; b < B; ++b) {
                const int cw = warp * 32 + (it0 + b) * RPI + sub;
                const float* x = xs[b];
                float mx = 0.f;
#pragma unroll
                for (int e = 0; e < 8; ++e) mx = fmaxf(mx, fabsf(x[e]));
#pragma unroll
                for (int o = CH / 2; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
                const int ex = min(max((int)(__float_as_uint(mx) >> 23) - 127, -100), 120);
                const float fac = __uint_as_float((uint32_t)(127 - ex) << 23);
                if (ch == 0) cmul[cw] = p.scale_log2 * __uint_as_float((uint32_t)(127 + ex) << 23);
                uint32_t hi[4], lo[4];
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const float a = x[2 * k] * fac, c = x[2 * k + 1] * fac;
                    const __half2 h = __floats2half2_rn(a, c);
                    const float2 f = __half22float2(h);
                    const __half2 r = __floats2half2_rn(a - f.x, c - f.y);
                    hi[k] = *reinterpret_cast<const uint32_t*>(&h);
                    lo[k] = *reinterpret_cast<const uint32_t*>(&r);
                }
                *reinterpret_cast<uint4*>(q_dst(cw, ch)) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
                *reinterpret_cast<uint4*>(q_dst(cw, ch) + QPART) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
            }
        }
    }
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    if (tid == 0) {
        dead = 0;
        any_odd = 0;
    }
    if (tid < kBulkMaxSplit / 32) odd[tid] = 0;
    const RowView view = row_view(p, my_len, my_seq, shared);
    if (live && split == 0 && view.n - view.shared > p.max_private) kv_flag(p.err, kKvBadPos);
    const int lim = live ? max(0, view.shared) : 0;
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    pdl_launch_dependents();  // the private items need nothing of this kernel
    const uint32_t tmem = tmem_at;
    const int t1 = min(lim_max, t0 + p.ls), seen_by_all = lim_min;
    const int nt = t0 < t1 ? (t1 - t0 + NK - 1) / NK : 0;  // 0: no column sees this far
    float* rows = reinterpret_cast<float*>(base);           // at the end: O's rows, [column][D + 4]
    float2* row_ml = reinterpret_cast<float2*>(base + bulk_rows_bytes(D, TILES));  // (m, l); l -1: padding
    if (nt > 0) {
    // S; then, in the place of each half of its positions, P hi (32 columns) and P lo (32)
    auto s_at = [&](int w) { return tmem + (uint32_t)(w * NK); };
    auto o_at = [&](int w) { return tmem + (uint32_t)(TILES * NK + w * D); };

    auto full = [&](int m) { return bulk_wait(&kv_full[m % NS], (uint32_t)(m / NS) & 1, &dead, p.err); };

    if (warp == LOADER) {
        int m = min(kBulkEarly, 2 * nt);  // (these are under way)
        for (; m < 2 * nt; ++m) {
            const bool ok = m < NS || bulk_wait(&kv_free[m % NS], (uint32_t)(m / NS - 1) & 1, &dead, p.err);
            if (!__all_sync(0xffffffffu, ok)) break;
            load(m, t1);
        }
        if (lane == 0 && dead)  // copies still in flight land before the CTA's memory is given up
            for (int q = max(0, m - NS); q < m; ++q) {
                const long long since = clock64();
                while (!mbar_try_wait(&kv_full[q % NS], (uint32_t)(q / NS) & 1) && clock64() - since < 200000000LL) {}
            }
    } else if (warp >= MMA) {
        // the column tiles this warp multiplies for: FP32, one each; binary16, the first warp both in turn
        const int w0 = F32 ? warp - MMA : 0, w1 = F32 ? min(w0 + 1, tiles) : warp == MMA ? tiles : 0;
        if (lane == 0 && w0 < w1) {
            constexpr uint32_t iqk = umma_idesc(NK, false), ipv = umma_idesc(D, true);
            auto qk = [&](int w, int j) {
                uint32_t ks = slot(2 * j), qa = smem_u32(base) + (uint32_t)(w * HN * QPART);
                asm volatile("" : "+r"(ks), "+r"(qa));  // (descriptors are formed here, not kept over the loop)
#pragma unroll
                for (int part = HN - 1; part >= 0; --part)  // lo, then hi
#pragma unroll
                    for (int k = 0; k < D / 16; ++k) {
                        const uint32_t off = (uint32_t)(k & 3) * 32;
                        tc_mma_ss(s_at(w), umma_desc(qa + part * QPART + (k >> 2) * (128 * 128) + off, 16, 1024),
                                  umma_desc(ks + (k >> 2) * (NK * 128) + off, 16, 1024), iqk, part != HN - 1 || k > 0);
                    }
                tc_commit(&s_full[w]);
                if (w == w1 - 1) tc_commit(&kv_free[2 * j % NS]);
            };
            auto pv = [&](int w, int j, int h) {
                uint32_t vs = slot(2 * j + 1);
                asm volatile("" : "+r"(vs));
#pragma unroll
                for (int part = HN - 1; part >= 0; --part)
#pragma unroll
                    for (int k = 0; k < NK / 32; ++k)
                        tc_mma_ts(o_at(w), s_at(w) + h * (NK / 2) + part * (NK / 4) + k * 8,
                                  umma_desc(vs + (h * (NK / 32) + k) * 2048, NK * 128, 1024), ipv,
                                  j > 0 || h > 0 || part != HN - 1 || k > 0);
                if (h == 0) tc_commit(&pv_half[w]);
            };
            bool ok = full(0);
            tc_fence_after();
            for (int w = w0; w < w1 && ok; ++w) qk(w, 0);
            for (int j = 0; j < nt && ok; ++j)
                for (int w = w0; w < w1 && ok; ++w) {
                    if (w == w0 && !(ok = full(2 * j + 1))) break;
                    for (int h = 0; h < 2 && ok; ++h) {
                        if (!(ok = bulk_wait(&p_ready[w][h], (uint32_t)j & 1, &dead, p.err))) break;
                        tc_fence_after();
                        pv(w, j, h);
                    }
                    if (!ok) break;
                    if (w == w1 - 1) tc_commit(&kv_free[(2 * j + 1) % NS]);
                    if (j + 1 < nt) {
                        if (w == w0 && !(ok = full(2 * j + 2))) break;
                        tc_fence_after();
                        qk(w, j + 1);
                    }
                }
            tc_commit(&o_done);  // after a failed wait too: whatever was issued ends before tensor memory is freed
        }
    } else if (wg < tiles) {
        const uint32_t lane_at = (uint32_t)(warp & 3) * 32u << 16;
        const uint32_t S = s_at(wg) + lane_at, O = o_at(wg) + lane_at;
        const float cm = fmaxf(cmul[tid], 1e-36f);  // (-inf * 0 would be NaN; below this every score is 0)
        const int wtid = tid & 127;
        float mref = 0.f, l = 0.f;
        bool ok = true;
        for (int j = 0; j < nt; ++j) {
            const int c0 = t0 + j * NK;
            const bool masked = c0 + NK > min(seen_by_all, t1);
            ok = __all_sync(0xffffffffu, bulk_wait(&s_full[wg], (uint32_t)j & 1, &dead, p.err));
            if (!ok) break;
            tc_fence_after();
            if (masked) {  // V where not every column sees: nothing but finite values may meet a zero weight
                full(2 * j + 1);
                uint8_t* V = ring + (size_t)((2 * j + 1) % NS) * SLOT;
                for (int k = wtid; k < NK * (D / 8); k += 128) {
                    const int r = k / (D / 8), ch = k % (D / 8), t = c0 + r;
                    if (t < seen_by_all && t < t1) continue;
                    uint4* w = reinterpret_cast<uint4*>(V + (ch >> 3) * (NK * 128) + r * 128 + (((ch & 7) ^ (r & 7)) << 4));
                    uint4 x = *w;
                    uint32_t* xs = reinterpret_cast<uint32_t*>(&x);
                    bool bad = false;
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        if ((xs[e] & 0x7c00u) == 0x7c00u) { xs[e] &= 0xffff0000u; bad = true; }
                        if ((xs[e] & 0x7c000000u) == 0x7c000000u) { xs[e] &= 0xffffu; bad = true; }
                    }
                    if (t >= t1) x = make_uint4(0, 0, 0, 0);
                    if (t >= t1 || bad) *w = x;
                    if (t < t1 && bad) {
                        atomicOr(&odd[(t - t0) >> 5], 1u << ((t - t0) & 31));
                        any_odd = 1;
                    }
                }
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            }
            uint64_t sum2[2] = {0, 0};
            const uint64_t cm2 = f2_pack(cm, cm), gain2 = f2_pack(kPaGain, kPaGain);
            uint32_t s[64];
            tc_ld32(S, s);
            tc_ld32(S + 32, s + 32);
#pragma unroll
            for (int h = 0; h < 2; ++h) {  // halves of 64 positions, each with its own look at the maximum
                tc_wait_ld();
                tc_loaded(s);
                tc_loaded(s + 32);
                if (masked) {
#pragma unroll
                    for (int e = 0; e < 64; ++e)
                        if (c0 + h * 64 + e >= lim) s[e] = 0xff800000u;  // -inf
                }
                float mx4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                for (int e = 0; e < 64; e += 2) mx4[(e >> 1) & 3] = max3(mx4[(e >> 1) & 3], __uint_as_float(s[e]), __uint_as_float(s[e + 1]));
                const float mx = max3(fmaxf(mx4[0], mx4[1]), mx4[2], mx4[3]) * cm;
                if (j == 0 && h == 0) {
                    mref = fmaxf(mx, kBulkLowest);  // (below any finite score, where none has been seen)
                } else if (__any_sync(0xffffffffu, mx > mref + kPaSlack)) {
                    const float next = fmaxf(mref, mx), corr = ex2(mref - next);
                    mref = next;
                    l *= corr;
                    sum2[0] = f2_mul(sum2[0], f2_pack(corr, corr));
                    sum2[1] = f2_mul(sum2[1], f2_pack(corr, corr));
                    // every product into O so far has to be complete: before S(j) the earlier tiles', before its
                    // second half the first half's
                    if (h == 1) {
                        ok = __all_sync(0xffffffffu, bulk_wait(&pv_half[wg], (uint32_t)j & 1, &dead, p.err));
                        tc_fence_after();
                    }
#pragma unroll 1
                    for (int k = 0; k < D; k += 16) {
                        uint32_t o[16];
                        tc_ld16(O + k, o);
#pragma unroll
                        for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * corr);
                        tc_st16(O + k, o);
                    }
                }
                // ---- the weights: binary16 rows carry the factor in the exponent (their rounding is 2^-11 anyway)
                const float shift = F32 ? -mref : 7.f - mref;
                const uint64_t sh2 = f2_pack(shift, shift);
#pragma unroll
                for (int k = 0; k < 64; k += 32) {
                    uint32_t hi[16], lo[F32 ? 16 : 1];
#pragma unroll
                    for (int e = 0; e < 16; ++e) {
                        float a, b;
                        f2_unpack(f2_fma(f2_pack(__uint_as_float(s[k + 2 * e]), __uint_as_float(s[k + 2 * e + 1])), cm2, sh2), a, b);
                        a = ex2(a);
                        b = ex2(b);
                        uint64_t ab = f2_pack(a, b);
                        sum2[e & 1] = f2_add(sum2[e & 1], ab);
                        if constexpr (F32) {
                            ab = f2_mul(ab, gain2);
                            f2_unpack(ab, a, b);
                        }
                        const __half2 x = __floats2half2_rn(a, b);
                        hi[e] = *reinterpret_cast<const uint32_t*>(&x);
                        if constexpr (F32) {
                            const float2 f = __half22float2(x);
                            const __half2 r = __floats2half2_rn(a - f.x, b - f.y);
                            lo[e] = *reinterpret_cast<const uint32_t*>(&r);
                        }
                    }
                    tc_st16(S + h * 64 + k / 2, hi);
                    if constexpr (F32) tc_st16(S + h * 64 + 32 + k / 2, lo);
                    if (h == 0) tc_ld32(S + 64 + k, s + k);  // the second half's scores take the used ones' registers
                }
                tc_wait_st();
                tc_fence_before();
                mbar_arrive(&p_ready[wg][h]);
            }
            if (!ok) break;
            float a, b;
            f2_unpack(f2_add(sum2[0], sum2[1]), a, b);
            l += a + b;
        }
        ok = __all_sync(0xffffffffu, bulk_wait(&o_done, 0, &dead, p.err)) && ok;
        tc_fence_after();
        named_sync(1, 128 * tiles);  // both tiles' notes of odd positions (every softmax warp comes here)
        if (ok) {
            // O's rows into shared memory, where the loads and Q are done with
#pragma unroll 1
            for (int k = 0; k < D; k += 32) {
                uint32_t o[32];
                tc_ld32(O + k, o);
                tc_wait_ld();
                tc_loaded(o);
                if (any_odd)
                    for (int t = t0; t < min(t1, lim); ++t)
                        if (odd[(t - t0) >> 5] >> ((t - t0) & 31) & 1) {
                            int id = page_ids[(t >> p.page_shift) - first_page];
                            if (id < 0 || id >= p.num_pages) id = 0;
                            const __half* v = p.vp + (((((size_t)id * p.kv_heads + kvh) << p.page_shift) +
                                                       (t & ((1 << p.page_shift) - 1))) * D + k);
#pragma unroll
                            for (int e = 0; e < 32; ++e) {
                                const float x = __half2float(v[e]);
                                if (!(fabsf(x) <= 65504.f)) o[e] = __float_as_uint(__uint_as_float(o[e]) + x);
                            }
                        }
                uint4* dst = reinterpret_cast<uint4*>(rows + (size_t)tid * (D + 4) + k);
#pragma unroll
                for (int e = 0; e < 8; ++e) dst[e] = make_uint4(o[4 * e], o[4 * e + 1], o[4 * e + 2], o[4 * e + 3]);
            }
            row_ml[tid] = make_float2(lim <= t0 || l == 0.f ? -INFINITY : mref, live && view.n < 0 ? -1.f : F32 ? l * kPaGain : l);
        }
        tc_fence_before();
    }
    __syncwarp();
    __syncthreads();
    if (warp == MMA) {
        if (lane == 0) bulk_wait(&o_done, 0, &dead, p.err);
        __syncwarp();
        tc_fence_after();
        tc_dealloc(tmem, 256 * TILES);
    }
    } else {
        if (warp == MMA) tc_dealloc(tmem, 256 * TILES);
        if (tid < 128 * tiles) row_ml[tid] = make_float2(-INFINITY, live && view.n < 0 ? -1.f : 0.f);
    }
    // ---- join the cluster's splits: CTA `rank` takes every C-th block of rows, a warp a row at a time
    // (a lane four dimensions), the splits' rows loaded together and added in split order
    if (C > 1) cluster.sync();
    else __syncthreads();
    constexpr int LPR = D / 4, RPW = 32 / LPR;  // lanes per row, rows per warp and step
    const int ns = p.nss + p.nsp, slot_at = split / C, cols = min(COLS, ncol - col0);
    bool odd_out = false;  // this thread has stored an output that is not finite
    auto join = [&](auto cc) {
        constexpr int CC = decltype(cc)::value, U = 8 / CC;  // U rows at a time: eight loads in flight
        const float* far_rows[CC];
        const float2* far_ml[CC];
#pragma unroll
        for (int c = 0; c < CC; ++c) {
            far_rows[c] = CC > 1 ? cluster.map_shared_rank(rows, c) : rows;
            far_ml[c] = CC > 1 ? cluster.map_shared_rank(row_ml, c) : row_ml;
        }
        constexpr int STEP = RPW * CC;
        const int e0 = lane % LPR * 4;
        for (int r = (warp * U * CC + rank) * RPW; r < cols; r += (bulk_threads(TILES) / 32) * U * STEP) {
            float2 ml[U][CC];
            float4 v[U][CC];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int cw = min(r + u * STEP + lane / LPR, cols - 1);
#pragma unroll
                for (int c = 0; c < CC; ++c) {
                    ml[u][c] = far_ml[c][cw];
                    v[u][c] = *reinterpret_cast<const float4*>(far_rows[c] + (size_t)cw * (D + 4) + e0);
                }
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int cw = r + u * STEP + lane / LPR;
                if (cw >= cols || ml[u][0].y < 0.f) continue;  // (negative: padding)
                float M = -INFINITY, L = 0.f;
#pragma unroll
                for (int c = 0; c < CC; ++c) M = fmaxf(M, ml[u][c].x);
                float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
                for (int c = 0; c < CC; ++c)
                    if (ml[u][c].x != -INFINITY) {
                        const float w = ex2(ml[u][c].x - M);
                        L = fmaf(ml[u][c].y, w, L);
                        a.x = fmaf(v[u][c].x, w, a.x); a.y = fmaf(v[u][c].y, w, a.y);
                        a.z = fmaf(v[u][c].z, w, a.z); a.w = fmaf(v[u][c].w, w, a.w);
                    }
                const int qr = row_of(cw);
                const size_t row = (size_t)(r0 + base_row + qr);
                const int head = kvh * p.G + cw + base_head - qr * p.G;
                if (p.direct) {
                    const float iv = M == -INFINITY ? 0.f : 1.f / L;
                    T* dst = static_cast<T*>(p.out) + row * p.ldo + (size_t)head * D + e0;
                    const float o[4] = {a.x * iv, a.y * iv, a.z * iv, a.w * iv};
                    if (p.out_vec) {
                        if constexpr (F32) {
                            *reinterpret_cast<float4*>(dst) = make_float4(o[0], o[1], o[2], o[3]);
                        } else {
                            const __half2 x = __floats2half2_rn(o[0], o[1]), y = __floats2half2_rn(o[2], o[3]);
                            *reinterpret_cast<uint2*>(dst) =
                                make_uint2(*reinterpret_cast<const uint32_t*>(&x), *reinterpret_cast<const uint32_t*>(&y));
                        }
                    } else {
#pragma unroll
                        for (int e = 0; e < 4; ++e) dst[e] = kv_out<T>(o[e]);
                    }
                    const float z = (a.x + a.y) + (a.z + a.w);
                    odd_out |= z - z != 0.f && L == L;
                } else {
                    const size_t at = (row * p.heads + head) * ns + slot_at;
                    *reinterpret_cast<float4*>(p.part_o + at * D + e0) = a;
                    if (e0 == 0) p.part_ml[at] = make_float2(M, L);
                }
            }
        }
    };
    if (C == 1) join(std::integral_constant<int, 1>{});
    else if (C == 2) join(std::integral_constant<int, 2>{});
    else if (C == 4) join(std::integral_constant<int, 4>{});
    else join(std::integral_constant<int, 8>{});
    if (odd_out) {  // (NaN: looked up, row by row as the join took them)
        const int take = 8 / C;
#pragma unroll 1
        for (int k = 0;; ++k) {
            const int cw = ((k / take * (bulk_threads(TILES) / 32) + warp) * take * C + rank + k % take * C) * RPW + lane / LPR;
            if (cw >= COLS) break;
            if (cw >= cols || row_ml[cw].y < 0.f) continue;
            const int qr = row_of(cw), row = r0 + base_row + qr;
            odd_outputs(p, row, kvh, D, lane % LPR * 4,
                        static_cast<T*>(p.out) + (size_t)row * p.ldo + (size_t)(kvh * p.G + cw + base_head - qr * p.G) * D + lane % LPR * 4, 4);
        }
    }
    if (C > 1) cluster.sync();  // no CTA leaves while another may still read its rows
    groupless_rows<D, T>(p);
}

}  // namespace laic
