// The serving operators' entry points: a KV cache in pages (append, attention),
// probabilities of logits rows and the verification of drafted tokens.
#include "serving.cuh"

#include <algorithm>
#include <atomic>
#include <climits>
#include <new>

#include "launch.cuh"
#include "paged.cuh"
#include "paged_attn.cuh"
#include "paged_bulk.cuh"
#include "verify.cuh"

namespace laic {
namespace {

// The pages' device for the call; the thread's current one afterwards.
struct DeviceGuard {
    int prev = -1;
    cudaError_t err = cudaSuccess;
    explicit DeviceGuard(int device) {
        int cur = -1;
        err = cudaGetDevice(&cur);
        if (err == cudaSuccess && cur != device) {
            err = cudaSetDevice(device);
            if (err == cudaSuccess) prev = cur;
        }
    }
    ~DeviceGuard() {
        if (prev >= 0) cudaSetDevice(prev);
    }
};

int cuda_fail(cudaError_t e, const char* what) {
    return api_fail(LAIC_E_CUDA, std::string(what) + ": " + cudaGetErrorString(e));
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }
bool type_ok(int t) { return t == LAIC_GGML_F32 || t == LAIC_GGML_F16; }
int type_size(int t) { return t == LAIC_GGML_F32 ? 4 : 2; }
int log2i(int v) {
    int s = 0;
    while ((1 << s) < v) ++s;
    return s;
}

int check_pages(const laic_kv_pages& g) {
    if (g.head_dim != 32 && g.head_dim != 64 && g.head_dim != 128)
        return api_fail(LAIC_E_UNSUPPORTED, "head_dim must be 32, 64 or 128");
    if (g.kv_heads < 1 || g.num_pages < 1) return api_fail(LAIC_E_INVALID, "kv_heads and num_pages must be >= 1");
    if (g.page_size < 16 || g.page_size > 256 || (g.page_size & (g.page_size - 1)))
        return api_fail(LAIC_E_UNSUPPORTED, "page_size must be 16, 32, 64, 128 or 256");
    return LAIC_OK;
}
int check_page_ptrs(const laic_kv_pages& g) {
    if (!g.k_dev || !g.v_dev || !g.err_dev) return api_fail(LAIC_E_INVALID, "null page or error pointer");
    if (!aligned16(g.k_dev) || !aligned16(g.v_dev)) return api_fail(LAIC_E_INVALID, "pages must be 16-byte aligned");
    return LAIC_OK;
}
int check_table(int rows, int nseq, int pages_per_seq, int page_size, const int32_t* seq) {
    if (nseq < 1 || pages_per_seq < 1) return api_fail(LAIC_E_INVALID, "nseq and pages_per_seq must be >= 1");
    if ((long long)pages_per_seq * page_size > INT_MAX) return api_fail(LAIC_E_INVALID, "page table row too long");
    if (!seq && nseq < rows) return api_fail(LAIC_E_INVALID, "without seq_dev every row needs its page table row");
    return LAIC_OK;
}

// Runs `f` (the launches of a checked call) on `device`.
template <typename F>
int on_device(int device, F&& f) {
    DeviceGuard dg(device);
    if (dg.err != cudaSuccess) return cuda_fail(dg.err, "device");
    return f();
}

// The result of a launch, counted where it was made. (With LaunchOpts::pdl every first kernel of a call may start
// while its predecessor in the stream drains; it waits before it reads or writes anything.)
cudaError_t counted(cudaError_t e, const LaunchOpts& o) {
    if (e == cudaSuccess && o.launches) ++*o.launches;
    return e;
}
template <typename TI, typename TQ>
cudaError_t append_launch(bool vec, dim3 grid, int block, cudaStream_t st, const LaunchOpts& o, const KvAppendParams& p) {
    void (*fn)(KvAppendParams) = vec ? kv_append_kernel<TI, TQ, true, 1> : kv_append_kernel<TI, TQ, false, 1>;
    if constexpr (sizeof(TI) == 2 && sizeof(TQ) == 2)
        if (grid.x < (unsigned)p.rows) fn = kv_append_kernel<TI, TQ, true, 2>;
    return counted(launch_k(fn, grid, dim3(block), 0, st, o.pdl, p), o);
}

int device_sms(int dev) {
    static std::atomic<int> sms[64];
    if (dev < 0 || dev >= 64) return 148;
    int n = sms[dev].load();
    if (!n) {
        if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || n <= 0) {
            cudaGetLastError();
            return 148;
        }
        sms[dev].store(n);
    }
    return n;
}

using BulkFn = void (*)(KvAttnParams, CUtensorMap, CUtensorMap);
template <int TILES>
BulkFn bulk_fn(int D, bool f32) {
    if (D == 64) return f32 ? paged_bulk_kernel<64, float, TILES> : paged_bulk_kernel<64, __half, TILES>;
    return f32 ? paged_bulk_kernel<128, float, TILES> : paged_bulk_kernel<128, __half, TILES>;
}
BulkFn bulk_pick(int D, bool f32, int tiles) { return tiles == 1 ? bulk_fn<1>(D, f32) : bulk_fn<2>(D, f32); }

// Clusters of c CTAs of a kernel that are resident at once on the current device, 0 where that cannot be asked.
template <typename K>
int resident_clusters(K kernel, int threads, size_t smem, int c, int sms) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(c * sms);
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = (unsigned)c;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    int n = 0;
    if (cudaOccupancyMaxActiveClusters(&n, kernel, &cfg) == cudaSuccess && n > 0) return n;
    cudaGetLastError();
    return 0;
}
// The same, asked once per device and size (`known` of the kernel); where it cannot be, per_sm CTAs on each SM.
template <typename K>
int known_clusters(std::atomic<int> (&known)[64][9], K kernel, int threads, size_t smem, int device, int c, int per_sm) {
    const int guess = per_sm * device_sms(device) / c;
    if (device < 0 || device >= 64) return guess;
    int n = known[device][c].load();
    if (n) return n;
    DeviceGuard dg(device);
    if (dg.err != cudaSuccess || serving_set_attributes() != cudaSuccess) {
        cudaGetLastError();
        return guess;
    }
    n = resident_clusters(kernel, threads, smem, c, device_sms(device));
    if (!n) return guess;
    known[device][c].store(n);
    return n;
}
int bulk_clusters(int device, int c) {  // (the largest's: a CTA takes an SM's tensor memory or shared memory)
    static std::atomic<int> known[64][9];
    return known_clusters(known, bulk_pick(128, true, 2), bulk_threads(2), bulk_smem(128, true, 2), device, c, 1);
}
int verify_clusters(int device, int c) {
    static std::atomic<int> known[64][9];
    return known_clusters(known, verify_kernel<true>, kVerifyThreads, 0, device, c, 2);
}
static_assert(kBulkMaxCluster <= 8 && kVerifyMaxCluster <= 8, "known_clusters' tables");
// ---- attention: how a call is cut into items
struct AttnPlan {
    int nt = 1;            // column tiles of 8 of a shared item
    int lp = 64, nsp = 1;  // private splits
    int ls = 64, nss = 0, ctiles = 0;
    int shared_items = 0, private_items = 0;
    bool bulk = false;     // the shared items run in paged_bulk.cuh,
    int mt = 1;            // M tiles per CTA there
    int cluster = 1;       // this many splits of a set of columns in a cluster (nss counts clusters)
    bool whole = false;    // a CTA per row and kv head finishes the row
    bool direct = false;   // the bulk kernel's clusters do
    size_t ml_off = 0, bytes = 0;
};

// A group goes to the bulk kernel from this many columns (query rows x heads per kv head) and shared positions on.
// Measured on 8 kv heads, 1 to 8 groups, 128 to 8,192 positions, us of the items / of the bulk kernel:
//   head_dim 64: 24 columns 34 / 42, 28: 54 / 42; with private positions, whose CTAs run beside items but not beside
//   bulk CTAs (which fill their SM), 32: 58 / 69, 64: 110 / 71;
//   head_dim 128: 16 columns 47 / 50 (FP32), 20: 60 / 50 and 52 / 37 (binary16);
//   128 positions: 32 columns 13 / 10 and 14 / 12; 64 positions at head_dim 128: 12 / 14.
int bulk_min_cols(int head_dim, bool has_private) { return head_dim == 128 ? 20 : has_private ? 40 : 28; }
constexpr int kBulkMinShared = 128;

int round_up(long long v, int m) { return (int)((v + m - 1) / m * m); }

constexpr int kMaxPositions = 1073000000;
static_assert(2LL * kMaxPositions + 16 * kBulkMaxCluster * kBulkMaxSplit <= INT_MAX, "positions past a row's end stay within an int");

int check_attention(const laic_kv_pages& g, const laic_kv_attention_args& a) {
    if (int rc = check_pages(g)) return rc;
    if (a.rows < 0) return api_fail(LAIC_E_INVALID, "rows must be >= 0");
    if (a.heads < 1 || a.heads % g.kv_heads) return api_fail(LAIC_E_INVALID, "heads must be a multiple of kv_heads");
    if (a.heads / g.kv_heads > 8) return api_fail(LAIC_E_UNSUPPORTED, "at most 8 query heads per kv head");
    if ((long long)a.rows * a.heads > INT_MAX) return api_fail(LAIC_E_UNSUPPORTED, "too many rows of heads");
    if (!type_ok(a.type)) return api_fail(LAIC_E_UNSUPPORTED, "query and output type must be F32 or F16");
    if (!(a.scale >= 0.f)) return api_fail(LAIC_E_INVALID, "scale must not be negative");
    if (a.max_len < 0 || a.groups < 0 || a.max_private < -1) return api_fail(LAIC_E_INVALID, "negative bound");
    if (a.groups && (a.max_group_rows < 1 || a.max_shared < 0 || a.max_group_rows > a.rows))
        return api_fail(LAIC_E_INVALID, "groups need max_group_rows in [1, rows] and max_shared >= 0");
    // (a shared length, a private one and a split added up stay within 32 bits)
    if (a.max_len > kMaxPositions || (a.groups && a.max_shared > kMaxPositions))
        return api_fail(LAIC_E_UNSUPPORTED, "max_len and max_shared must not exceed 1,073,000,000 positions");
    const long long cap = (long long)a.pages_per_seq * g.page_size;
    if (a.max_len > cap || (a.groups && a.max_shared > cap))
        return api_fail(LAIC_E_INVALID, "max_len and max_shared must not exceed pages_per_seq * page_size");
    return LAIC_OK;
}

int plan_attention(const laic_kv_pages& g, const laic_kv_attention_args& a, AttnPlan& pl) {
    const int G = a.heads / g.kv_heads;
    const int max_private = a.max_private < 0 ? a.max_len : std::min(a.max_private, a.max_len);
    // splits of `len` positions over `pairs` items each: about `want` items; a range of up to `whole` stays in
    // one piece and none is shorter than 128 (a join costs more than that many positions)
    auto split = [&](long long pairs, int len, long long want, int unit, int whole, int most) {
        if (len <= whole) return round_up(std::max(len, 1), unit);
        const long long l = std::min<long long>(((long long)len * pairs + want - 1) / want, kMaxPositions);
        return std::max(128, std::min(round_up(l, unit), most));
    };
    const int sms = device_sms(g.device);
    // private: short ranges by one CTA, which writes the output; longer ones by a warp per split, 8 to 12 on an SM
    // (256 positions: a partial costs 2 % of their bytes, and ragged rows balance; more where the bound is far,
    // which would ask for thousands of partials per row).
    // A CTA's warps walk a range of 1,024 in 16 to 25 us whatever the rows; splits and their merge take 9 to 14 for
    // 64 (row, kv head) pairs, but 62 against 45 for 512: they meet near 448 positions, or 370 pairs.
    const bool many = 2LL * a.rows * g.kv_heads >= 5LL * sms;
    const int cols = a.max_group_rows * G;
    pl.bulk = a.groups && g.head_dim >= 64 && cols >= bulk_min_cols(g.head_dim, max_private > 0) &&
              a.max_shared >= kBulkMinShared && (long long)g.num_pages * g.kv_heads * g.page_size <= INT_MAX;
    pl.whole = max_private <= (many ? kPrWhole : 448);
    const int most = std::max(256, std::min(kPrWhole, max_private / 64 / 16 * 16));
    pl.lp = pl.whole ? kPrWhole : split((long long)a.rows * g.kv_heads, max_private, 12LL * sms, 16, 128, most);
    pl.nsp = pl.whole ? 0 : (max_private + pl.lp - 1) / pl.lp;
    if (a.groups) {
        if (max_private == 0) pl.whole = false;  // nothing private: shared items alone, joined by the merge
        if (pl.bulk) {
            // about one CTA per SM (a bulk CTA fills one), in whole tiles, as few clusters per set of columns
            // as that allows
            pl.mt = cols <= 128 ? 1 : kBulkTiles;
            pl.ctiles = (cols + bulk_cols(pl.mt) - 1) / bulk_cols(pl.mt);
            const long long sets = (long long)a.groups * pl.ctiles * g.kv_heads;
            const long long splits = std::max(1LL, (a.max_shared + 2LL * kBulkKeys - 1) / (2 * kBulkKeys));  // two tiles each
            int best = 1, count = 1;
            for (int c = kBulkMaxCluster; c >= 1; c /= 2) {
                const long long fit = std::min(bulk_clusters(g.device, c) / sets, (splits + c - 1) / c);
                if (c <= 2 * splits && fit * c > (long long)best * count) {
                    best = c;
                    count = (int)fit;
                }
            }
            pl.cluster = best;
            pl.ls = std::min(kBulkMaxSplit, std::max(2 * kBulkKeys, round_up((a.max_shared + best * count - 1) / (best * count), kBulkKeys)));
            pl.nss = (int)((a.max_shared + (long long)pl.ls * best - 1) / ((long long)pl.ls * best));
        } else {
            pl.nt = cols <= 24 ? (cols + 7) / 8 : 4;
            pl.ctiles = (cols + 8 * pl.nt - 1) / (8 * pl.nt);
            pl.ls = split((long long)a.groups * pl.ctiles * g.kv_heads, a.max_shared, 4LL * sms, kPaChunk, 256, 512);
            pl.nss = (a.max_shared + pl.ls - 1) / pl.ls;
        }
    }
    const long long si = (long long)a.groups * pl.ctiles * g.kv_heads * pl.nss * pl.cluster;
    const long long pi = (long long)a.rows * g.kv_heads * (pl.whole ? 1 : pl.nsp);
    if (si + pi > INT_MAX - kPrWarps) return api_fail(LAIC_E_UNSUPPORTED, "too many attention items");
    pl.shared_items = (int)si;
    pl.private_items = (int)pi;
    pl.direct = pl.bulk && pl.nss == 1 && pi == 0;
    if (!pl.direct && pl.nss + pl.nsp) {
        const size_t parts = (size_t)a.rows * a.heads * (pl.nss + pl.nsp);
        pl.ml_off = parts * g.head_dim * 4;
        pl.bytes = pl.ml_off + parts * 8;
    }
    return LAIC_OK;
}

using PaFn = void (*)(KvAttnParams);
template <int D, typename T>
PaFn pa_fn_nt(int nt) {
    return nt == 1   ? paged_attn_kernel<D, 1, T>
           : nt == 2 ? paged_attn_kernel<D, 2, T>
           : nt == 3 ? paged_attn_kernel<D, 3, T>
                     : paged_attn_kernel<D, 4, T>;
}
template <typename T>
PaFn pa_fn(int D, int nt) {
    return D == 32 ? pa_fn_nt<32, T>(nt) : D == 64 ? pa_fn_nt<64, T>(nt) : pa_fn_nt<128, T>(nt);
}
PaFn pa_pick(int D, int nt, int type) { return type == LAIC_GGML_F32 ? pa_fn<float>(D, nt) : pa_fn<__half>(D, nt); }
template <typename T, bool PK, bool WHOLE>
PaFn pr_fn(int D) {
    return D == 32   ? paged_private_kernel<32, T, PK, WHOLE>
           : D == 64 ? paged_private_kernel<64, T, PK, WHOLE>
                     : paged_private_kernel<128, T, PK, WHOLE>;
}
template <bool WHOLE>
PaFn pr_fn_type(int D, int type, int G) {
    return type == LAIC_GGML_F16 ? pr_fn<__half, false, WHOLE>(D) : G <= 4 ? pr_fn<float, true, WHOLE>(D) : pr_fn<float, false, WHOLE>(D);
}
PaFn pr_pick(int D, int type, int G, bool whole) { return whole ? pr_fn_type<true>(D, type, G) : pr_fn_type<false>(D, type, G); }
template <typename T>
PaFn pm_fn(int D) {
    return D == 32 ? paged_merge_kernel<32, T> : D == 64 ? paged_merge_kernel<64, T> : paged_merge_kernel<128, T>;
}

using EncodeFn = decltype(&cuTensorMapEncodeTiled);
EncodeFn tensor_map_encode() {
    static std::atomic<EncodeFn> fn{nullptr};
    EncodeFn f = fn.load();
    if (!f) {
        void* at = nullptr;
        cudaDriverEntryPointQueryResult found;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &at, cudaEnableDefault, &found) == cudaSuccess &&
            found == cudaDriverEntryPointSuccess)
            fn.store(f = reinterpret_cast<EncodeFn>(at));
    }
    return f;
}
// One pool as rows of head_dim binary16 values; a box is 64 columns (x 0 or 64: whole 128-byte lines) of
// up to a page's positions, so it never leaves a (page, head) run.
bool encode_pages(const laic_kv_pages& g, void* pool, CUtensorMap* map) {
    const EncodeFn f = tensor_map_encode();
    if (!f) return false;
    const cuuint64_t dims[2] = {(cuuint64_t)g.head_dim, (cuuint64_t)g.num_pages * g.kv_heads * g.page_size};
    const cuuint64_t strides[1] = {(cuuint64_t)g.head_dim * 2};
    const cuuint32_t box[2] = {64, (cuuint32_t)std::min(g.page_size, kBulkKeys)}, step[2] = {1, 1};
    return f(map, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 2, pool, dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE,
             CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

}  // namespace

cudaError_t serving_set_attributes() {
    static std::atomic<bool> done[64];
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    if (dev >= 0 && dev < 64 && done[dev].load()) return cudaSuccess;
    for (int D : {32, 64, 128})
        for (int nt : {1, 2, 3, 4})
            for (int type : {LAIC_GGML_F32, LAIC_GGML_F16}) {
                e = cudaFuncSetAttribute(pa_pick(D, nt, type), cudaFuncAttributeMaxDynamicSharedMemorySize,
                                         (int)pa_smem(D, nt, type == LAIC_GGML_F32));
                if (e != cudaSuccess) return e;
            }
    for (int D : {32, 64, 128})
        for (bool whole : {false, true})
            for (PaFn fn : {pr_pick(D, LAIC_GGML_F16, 1, whole), pr_pick(D, LAIC_GGML_F32, 4, whole), pr_pick(D, LAIC_GGML_F32, 8, whole)}) {
                e = cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)pr_smem(D));
                if (e != cudaSuccess) return e;
            }
    for (int D : {64, 128})
        for (bool f32 : {false, true}) {
            for (int mt = 1; mt <= kBulkTiles; ++mt) {
                e = cudaFuncSetAttribute(bulk_pick(D, f32, mt), cudaFuncAttributeMaxDynamicSharedMemorySize, bulk_smem(D, f32, mt));
                if (e != cudaSuccess) return e;
            }
        }
    for (auto fn : {probs_kernel<true, true>, probs_kernel<true, false>}) {
        e = cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, kProbsSlice * 4);
        if (e != cudaSuccess) return e;
    }
    if (dev >= 0 && dev < 64) done[dev].store(true);
    return cudaSuccess;
}

static_assert(kKvBadSeq == LAIC_KV_BAD_SEQ && kKvBadPos == LAIC_KV_BAD_POS && kKvBadPage == LAIC_KV_BAD_PAGE &&
              kKvBadGroup == LAIC_KV_BAD_GROUP && kKvWait == LAIC_KV_WAIT, "the public bits");

int kv_append(const laic_kv_pages& g, const laic_kv_append_args& a, cudaStream_t st, LaunchOpts o) {
    if (int rc = check_pages(g)) return rc;
    if (a.rows < 0 || a.heads < 0) return api_fail(LAIC_E_INVALID, "rows and heads must be >= 0");
    if (!type_ok(a.in_type) || !type_ok(a.q_type)) return api_fail(LAIC_E_UNSUPPORTED, "q, k and v must be F32 or F16");
    if (a.rope_dim < 0 || a.rope_dim > g.head_dim || (a.rope_dim & 1)) return api_fail(LAIC_E_INVALID, "invalid RoPE dimension");
    if (int rc = check_table(a.rows, a.nseq, a.pages_per_seq, g.page_size, a.seq_dev)) return rc;
    if (a.rows == 0) return LAIC_OK;
    if (int rc = check_page_ptrs(g)) return rc;
    if (!a.k_dev || !a.v_dev || !a.pos_dev || !a.page_table_dev || (a.heads && (!a.q_dev || !a.q_out_dev)))
        return api_fail(LAIC_E_INVALID, "null pointer");
    if (a.rope_dim && (!a.rope_dev || a.rope_positions < 1)) return api_fail(LAIC_E_INVALID, "rotation without a table");
    if ((reinterpret_cast<uintptr_t>(a.rope_dev) & 7) && a.rope_dim) return api_fail(LAIC_E_INVALID, "rotation table must be 8-byte aligned");
    const long long kvw = (long long)g.kv_heads * g.head_dim, qw = (long long)a.heads * g.head_dim;
    if (a.rows > 1 && (a.ldk < kvw || a.ldv < kvw || (a.heads && (a.ldq < qw || a.ldqo < qw))))
        return api_fail(LAIC_E_INVALID, "row strides must not be below the rows' widths");
    if (a.q_out_dev == a.q_dev && a.heads && (a.in_type != a.q_type || (a.rows > 1 && a.ldq != a.ldqo)))
        return api_fail(LAIC_E_INVALID, "rotation in place needs one type and stride");
    if (qw + 2 * kvw > INT_MAX) return api_fail(LAIC_E_UNSUPPORTED, "rows too wide");
    KvAppendParams p{};
    p.q = a.q_dev; p.k = a.k_dev; p.v = a.v_dev; p.q_out = a.q_out_dev;
    p.ldq = a.ldq; p.ldk = a.ldk; p.ldv = a.ldv; p.ldqo = a.ldqo;
    p.kp = static_cast<__half*>(g.k_dev); p.vp = static_cast<__half*>(g.v_dev);
    p.rows = a.rows; p.heads = a.heads; p.kv_heads = g.kv_heads; p.head_dim = g.head_dim;
    p.page_shift = log2i(g.page_size); p.num_pages = g.num_pages;
    p.pos = a.pos_dev; p.seq = a.seq_dev; p.table = a.page_table_dev;
    p.nseq = a.nseq; p.pages_per_seq = a.pages_per_seq;
    p.rope = reinterpret_cast<const float2*>(a.rope_dev);
    p.rope_pairs = a.rope_dim / 2; p.rope_positions = a.rope_dim ? a.rope_positions : INT_MAX;
    p.err = g.err_dev;
    const int bi = type_size(a.in_type), bq = type_size(a.q_type);
    const bool vec = aligned16(a.k_dev) && aligned16(a.v_dev) && a.ldk * bi % 16 == 0 && a.ldv * bi % 16 == 0 &&
                     (!a.heads || (aligned16(a.q_dev) && aligned16(a.q_out_dev) && a.ldq * bi % 16 == 0 && a.ldqo * bq % 16 == 0));
    p.vec_rope = a.rope_dim % 4 == 0 && aligned16(a.rope_dev);
    const int units = (a.heads + 2 * g.kv_heads) * (g.head_dim / 8);
    p.units = units;
    const int block = std::min(256, (units + 31) / 32 * 32), cta = block * kAppendUnits;
    // two rows per CTA of binary16 in and out from 40 rows per SM on (8,192 rows of 32 + 16 heads of 128: 37.5 us
    // against 38.5; 4,096: 19.0 against 18.7; FP32 on either side has the bytes in flight with one: 59 against 69)
    const bool two = vec && bi == 2 && bq == 2 && a.rows >= 40 * device_sms(g.device);
    const dim3 grid(two ? (a.rows + 1) / 2 : a.rows, (units + cta - 1) / cta);
    if (grid.y > 65535) return api_fail(LAIC_E_UNSUPPORTED, "rows too wide");
    return on_device(g.device, [&]() -> int {
        const bool i32 = a.in_type == LAIC_GGML_F32, q32 = a.q_type == LAIC_GGML_F32;
        const cudaError_t e = i32 ? (q32 ? append_launch<float, float>(vec, grid, block, st, o, p) : append_launch<float, __half>(vec, grid, block, st, o, p))
                                  : (q32 ? append_launch<__half, float>(vec, grid, block, st, o, p) : append_launch<__half, __half>(vec, grid, block, st, o, p));
        return e == cudaSuccess ? LAIC_OK : cuda_fail(e, "kv_append");
    });
}

int kv_attention_bytes(const laic_kv_pages& g, const laic_kv_attention_args& a, uint64_t* bytes) {
    AttnPlan pl;
    if (int rc = check_attention(g, a)) return rc;
    if (a.rows > 0)
        if (int rc = plan_attention(g, a, pl)) return rc;
    *bytes = pl.bytes;
    return LAIC_OK;
}

int kv_attention(const laic_kv_pages& g, const laic_kv_attention_args& a, cudaStream_t st, LaunchOpts o) {
    if (int rc = check_attention(g, a)) return rc;
    if (int rc = check_table(a.rows, a.nseq, a.pages_per_seq, g.page_size, a.seq_dev)) return rc;
    if (a.rows == 0) return LAIC_OK;
    if (int rc = check_page_ptrs(g)) return rc;
    if (!a.q_dev || !a.out_dev || !a.len_dev || !a.page_table_dev || (a.groups && (!a.group_rows_dev || !a.group_len_dev)))
        return api_fail(LAIC_E_INVALID, "null pointer");
    const long long qw = (long long)a.heads * g.head_dim;
    if (a.rows > 1 && (a.ldq < qw || a.ldo < qw)) return api_fail(LAIC_E_INVALID, "row strides must not be below the rows' widths");
    AttnPlan pl;
    if (int rc = plan_attention(g, a, pl)) return rc;
    if (pl.bytes && (!a.workspace_dev || a.workspace_bytes < pl.bytes))
        return api_fail(LAIC_E_INVALID, "laic_kv_attention needs " + std::to_string(pl.bytes) + " bytes of workspace");
    if (pl.bytes && !aligned16(a.workspace_dev)) return api_fail(LAIC_E_INVALID, "the workspace must be 16-byte aligned");
    KvAttnParams p{};
    p.q = a.q_dev; p.out = a.out_dev; p.ldq = a.ldq; p.ldo = a.ldo;
    p.kp = static_cast<const __half*>(g.k_dev); p.vp = static_cast<const __half*>(g.v_dev);
    p.num_pages = g.num_pages; p.page_shift = log2i(g.page_size);
    p.kv_heads = g.kv_heads; p.heads = a.heads; p.G = a.heads / g.kv_heads;
    p.g_inv = (65536 + p.G - 1) / p.G;
    p.len = a.len_dev; p.seq = a.seq_dev; p.table = a.page_table_dev;
    p.nseq = a.nseq; p.pages_per_seq = a.pages_per_seq; p.rows = a.rows; p.max_len = a.max_len;
    p.groups = a.groups; p.max_group_rows = a.max_group_rows; p.max_shared = a.max_shared;
    p.max_private = a.max_private < 0 ? a.max_len : std::min(a.max_private, a.max_len);
    p.group_rows = a.group_rows_dev; p.group_len = a.group_len_dev;
    const float scale = a.scale != 0.f ? a.scale : 1.f / sqrtf((float)g.head_dim);
    p.scale_log2 = scale * 1.44269504f;
    p.lp = pl.lp; p.nsp = pl.nsp; p.ls = pl.ls; p.nss = pl.nss; p.ctiles = pl.ctiles; p.lc = pl.cluster;
    p.private_items = pl.private_items;
    p.first = pl.shared_items == 0;
    p.direct = pl.direct;
    p.out_vec = aligned16(a.out_dev) && (a.rows == 1 || a.ldo * type_size(a.type) % 16 == 0);
    p.q_vec = aligned16(a.q_dev) && (a.rows == 1 || a.ldq * type_size(a.type) % 16 == 0);
    if (pl.bytes) {
        p.part_o = static_cast<float*>(a.workspace_dev);
        p.part_ml = reinterpret_cast<float2*>(static_cast<char*>(a.workspace_dev) + pl.ml_off);
    }
    p.err = g.err_dev;
    const bool f32 = a.type == LAIC_GGML_F32;
    return on_device(g.device, [&]() -> int {
        cudaError_t e = serving_set_attributes();
        if (e == cudaSuccess && pl.bulk && pl.shared_items) {
            CUtensorMap mk, mv;
            if (!encode_pages(g, g.k_dev, &mk) || !encode_pages(g, g.v_dev, &mv))
                return api_fail(LAIC_E_CUDA, "kv_attention: tensor map");
            e = counted(launch_cluster_k(bulk_pick(g.head_dim, f32, pl.mt), dim3(pl.shared_items), dim3(bulk_threads(pl.mt)),
                                         bulk_smem(g.head_dim, f32, pl.mt), st, o.pdl, pl.cluster, p, mk, mv), o);
        }
        if (e == cudaSuccess && !pl.bulk && pl.shared_items)
            e = counted(launch_k(pa_pick(g.head_dim, pl.nt, a.type), dim3(pl.shared_items), dim3(kPaWarps * 32),
                                 pa_smem(g.head_dim, pl.nt, f32), st, o.pdl, p), o);
        if (e == cudaSuccess && pl.private_items)
            e = counted(launch_k(pr_pick(g.head_dim, a.type, p.G, pl.whole),
                                 dim3(pl.whole ? pl.private_items : (pl.private_items + kPrWarps - 1) / kPrWarps),
                                 dim3(kPrWarps * 32), pr_smem(g.head_dim), st, o.pdl, p), o);
        if (e == cudaSuccess && !pl.direct && !pl.whole)
            e = counted(launch_k(f32 ? pm_fn<float>(g.head_dim) : pm_fn<__half>(g.head_dim),
                                 dim3((unsigned)(a.rows * a.heads)), dim3(kPmWarps * 32), 0,
                                 st, o.pdl && (pl.shared_items || pl.private_items), p), o);
        return e == cudaSuccess ? LAIC_OK : cuda_fail(e, "kv_attention");
    });
}

constexpr int kMaxVocab = 1 << 30;  // (the kernels step past a row's end by less than that, in an int)

int logits_probs(int device, int rows, int vocab, const float* x, long long ldx, const float* temp, float* y, long long ldy,
                 cudaStream_t st, LaunchOpts o) {
    if (rows < 0 || vocab < 1) return api_fail(LAIC_E_INVALID, "rows must be >= 0 and vocab >= 1");
    if (rows > INT_MAX / 8) return api_fail(LAIC_E_UNSUPPORTED, "too many rows");
    if (vocab > kMaxVocab) return api_fail(LAIC_E_UNSUPPORTED, "a vocabulary of at most 2^30");
    if (rows == 0) return LAIC_OK;
    if (!x || !temp || !y) return api_fail(LAIC_E_INVALID, "null pointer");
    if (rows > 1 && (ldx < vocab || ldy < vocab)) return api_fail(LAIC_E_INVALID, "row strides must not be below the vocabulary");
    if (x == y && rows > 1 && ldx != ldy) return api_fail(LAIC_E_INVALID, "in place needs one stride");
    ProbsParams p{x, y, temp, ldx, ldy, vocab};
    return on_device(device, [&]() -> int {
        const bool vec = aligned16(x) && aligned16(y) && (rows == 1 || (ldx % 4 == 0 && ldy % 4 == 0));
        // the smallest cluster whose shared memory holds the row; for few rows of some length the largest, to spread
        // them over the SMs (8 rows of 16,384: 4.4 us against 5.6; of 10,000: 4.3 against 4.5; of 8,192: 4.1 against 3.8)
        int c = 1;
        while (c < 8 && c * kProbsSlice < vocab) c *= 2;
        if (vocab >= 10000 && 8LL * rows <= device_sms(device)) c = 8;
        const bool sm = (long long)c * kProbsSlice >= vocab;
        if (!sm) c = 1;
        const auto fn = sm ? (vec ? probs_kernel<true, true> : probs_kernel<true, false>) : probs_kernel<false, false>;
        const size_t smem = sm ? ((((size_t)vocab + c - 1) / c + 3) & ~(size_t)3) * 4 : 0;
        cudaError_t e = serving_set_attributes();
        if (e == cudaSuccess)
            e = counted(launch_cluster_k(fn, dim3((unsigned)rows * c), dim3(kProbsThreads), smem, st, o.pdl, c, p), o);
        return e == cudaSuccess ? LAIC_OK : cuda_fail(e, "logits_probs");
    });
}

int verify_drafts(int device, const laic_verify_args& a, cudaStream_t st, LaunchOpts o) {
    if (a.nseq < 0 || a.vocab < 1) return api_fail(LAIC_E_INVALID, "nseq must be >= 0 and vocab >= 1");
    if (a.max_draft < 0) return api_fail(LAIC_E_INVALID, "max_draft must be >= 0");
    if (a.max_draft > LAIC_MAX_DRAFT) return api_fail(LAIC_E_UNSUPPORTED, "at most 64 drafted tokens per sequence");
    if (a.vocab > kMaxVocab) return api_fail(LAIC_E_UNSUPPORTED, "a vocabulary of at most 2^30");
    if (a.nseq > INT_MAX / kVerifyMaxCluster) return api_fail(LAIC_E_UNSUPPORTED, "too many sequences");
    if (a.nseq == 0) return LAIC_OK;
    if (!a.target_dev || !a.n_draft_dev || !a.sample_u_dev || !a.out_ids_dev || !a.out_n_dev ||
        (a.max_draft && (!a.draft_ids_dev || !a.accept_u_dev)))
        return api_fail(LAIC_E_INVALID, "null pointer");
    if (a.ld_target < a.vocab || (a.draft_dev && a.ld_draft < a.vocab))
        return api_fail(LAIC_E_INVALID, "row strides must not be below the vocabulary");
    VerifyParams p{a.target_dev, a.draft_dev, a.ld_target, a.ld_draft, a.draft_ids_dev, a.n_draft_dev, a.accept_u_dev,
                   a.sample_u_dev, a.out_ids_dev, a.out_n_dev, a.nseq, a.max_draft, a.vocab};
    return on_device(device, [&]() -> int {
        const bool vec = aligned16(a.target_dev) && a.ld_target % 4 == 0 &&
                         (!a.draft_dev || (aligned16(a.draft_dev) && a.ld_draft % 4 == 0));
        // the largest cluster of which all fit at once (vocabulary 128,256: 32 sequences in clusters of 8, 4, 2 take
        // 11.6, 13.0, 19.8 us, 36 take 17.9, 14.2, 19.5, 72 take 28, 25, 21)
        int c = kVerifyMaxCluster;
        while (c > 1 && a.nseq > verify_clusters(device, c)) c /= 2;
        const cudaError_t e = counted(launch_cluster_k(vec ? verify_kernel<true> : verify_kernel<false>, dim3((unsigned)a.nseq * c),
                                                       dim3(kVerifyThreads), 0, st, o.pdl, c, p), o);
        return e == cudaSuccess ? LAIC_OK : cuda_fail(e, "verify_drafts");
    });
}

}  // namespace laic

using laic::api_fail;

// No exception crosses the C boundary (the checks' messages allocate).
template <typename F>
static int guarded(F&& f) {
    try {
        return f();
    } catch (const std::bad_alloc&) {
        return LAIC_E_INVALID;
    }
}

extern "C" {

int laic_kv_append(const laic_kv_pages* pages, const laic_kv_append_args* args, void* stream) {
    return guarded([&] {
        if (!pages || !args) return api_fail(LAIC_E_INVALID, "null argument");
        return laic::kv_append(*pages, *args, (cudaStream_t)stream);
    });
}

int laic_kv_attention(const laic_kv_pages* pages, const laic_kv_attention_args* args, void* stream) {
    return guarded([&] {
        if (!pages || !args) return api_fail(LAIC_E_INVALID, "null argument");
        return laic::kv_attention(*pages, *args, (cudaStream_t)stream);
    });
}

int laic_kv_attention_workspace(const laic_kv_pages* pages, const laic_kv_attention_args* args, uint64_t* bytes) {
    return guarded([&] {
        if (!pages || !args || !bytes) return api_fail(LAIC_E_INVALID, "null argument");
        return laic::kv_attention_bytes(*pages, *args, bytes);
    });
}

int laic_kv_check(const laic_kv_pages* pages, void* stream) {
    return guarded([&] {
        if (!pages || !pages->err_dev) return api_fail(LAIC_E_INVALID, "null argument");
        return laic::on_device(pages->device, [&]() -> int {
            const cudaStream_t st = (cudaStream_t)stream;
            int bits = 0;
            cudaError_t e = cudaMemcpyAsync(&bits, pages->err_dev, 4, cudaMemcpyDeviceToHost, st);
            if (e == cudaSuccess) e = cudaStreamSynchronize(st);
            if (e == cudaSuccess && bits) e = cudaMemsetAsync(pages->err_dev, 0, 4, st);
            if (e == cudaSuccess && bits) e = cudaStreamSynchronize(st);
            if (e != cudaSuccess) return laic::cuda_fail(e, "laic_kv_check");
            return bits ? api_fail(LAIC_E_INVALID, laic::kv_error_text(bits)) : LAIC_OK;
        });
    });
}

int laic_logits_probs(int32_t device, int32_t rows, int32_t vocab, const float* logits_dev, int64_t ld_logits,
                      const float* temperature_dev, float* probs_dev, int64_t ld_probs, void* stream) {
    return guarded([&] {
        return laic::logits_probs(device, rows, vocab, logits_dev, ld_logits, temperature_dev, probs_dev, ld_probs,
                                  (cudaStream_t)stream);
    });
}

int laic_verify_drafts(int32_t device, const laic_verify_args* args, void* stream) {
    return guarded([&] {
        if (!args) return api_fail(LAIC_E_INVALID, "null argument");
        return laic::verify_drafts(device, *args, (cudaStream_t)stream);
    });
}

}  // extern "C"
