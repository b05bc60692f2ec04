// The serving operators' launches on a machine without a GPU: the runtime's calls are replaced by stand-ins that
// record each launch, and the checked entry points run as they are. A query per line,
//   append | attention rows heads max_len groups max_group_rows max_shared max_private | probs | verify   pdl
//   -> launches counted by the operator, then per recorded launch 1 where it may start early, else 0
#include <cuda.h>
#include <cuda_runtime.h>

#include <cstdio>
#include <iostream>
#include <sstream>
#include <string>
#include <vector>

static std::vector<int> early;
template <typename... A>
cudaError_t fake_launch(const cudaLaunchConfig_t* cfg, A&&...) {
    int e = 0;
    for (unsigned i = 0; i < cfg->numAttrs; ++i)
        if (cfg->attrs[i].id == cudaLaunchAttributeProgrammaticStreamSerialization)
            e = cfg->attrs[i].val.programmaticStreamSerializationAllowed;
    early.push_back(e);
    return cudaSuccess;
}
static CUresult fake_encode(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                            const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                            CUtensorMapL2promotion, CUtensorMapFloatOOBfill) {
    return CUDA_SUCCESS;
}
static cudaError_t fake_entry(const char*, void** at, unsigned long long, cudaDriverEntryPointQueryResult* found) {
    *at = reinterpret_cast<void*>(&fake_encode);
    *found = cudaDriverEntryPointSuccess;
    return cudaSuccess;
}
static cudaError_t fake_device(int* d) { *d = 0; return cudaSuccess; }
static cudaError_t fake_sms(int* n, cudaDeviceAttr, int) { *n = 148; return cudaSuccess; }
#define cudaLaunchKernelEx(...) fake_launch(__VA_ARGS__)
#define cudaGetDevice(d) fake_device(d)
#define cudaDeviceGetAttribute(n, a, d) fake_sms(n, a, d)
#define cudaFuncSetAttribute(...) cudaSuccess
#define cudaOccupancyMaxActiveClusters(n, ...) (*(n) = 16, cudaSuccess)
#define cudaGetDriverEntryPoint(...) fake_entry(__VA_ARGS__)
#include "serving.cu"

int laic::api_fail(int code, const std::string& msg) {
    std::fprintf(stderr, "%s\n", msg.c_str());
    return code;
}

int main() {
    std::string line, what;
    while (std::getline(std::cin, line)) {
        std::istringstream in(line);
        in >> what;
        void* const ptr = reinterpret_cast<void*>(4096);
        const laic_kv_pages pages{0, 2, 64, 64, 1000, ptr, ptr, (int32_t*)ptr};
        int n = 0, pdl = 0, rc = 0;
        early.clear();
        if (what == "append") {
            in >> pdl;
            laic_kv_append_args a{};
            a.rows = 3; a.heads = 8; a.nseq = 3; a.pages_per_seq = 100;
            a.ldq = a.ldqo = 512; a.ldk = a.ldv = 128;
            a.q_dev = a.k_dev = a.v_dev = a.q_out_dev = ptr;
            a.pos_dev = a.page_table_dev = (int32_t*)ptr;
            rc = laic::kv_append(pages, a, nullptr, {pdl != 0, &n});
        } else if (what == "attention") {
            laic_kv_attention_args a{};
            in >> a.rows >> a.heads >> a.max_len >> a.groups >> a.max_group_rows >> a.max_shared >> a.max_private >> pdl;
            a.nseq = a.rows; a.pages_per_seq = 100; a.ldq = a.ldo = a.heads * 64;
            a.q_dev = a.out_dev = ptr;
            a.len_dev = a.page_table_dev = a.group_rows_dev = a.group_len_dev = (int32_t*)ptr;
            a.workspace_dev = ptr; a.workspace_bytes = 1ull << 40;
            rc = laic::kv_attention(pages, a, nullptr, {pdl != 0, &n});
        } else if (what == "probs") {
            in >> pdl;
            rc = laic::logits_probs(0, 4, 50000, (float*)ptr, 50000, (float*)ptr, (float*)ptr, 50000, nullptr, {pdl != 0, &n});
        } else {
            in >> pdl;
            laic_verify_args a{};
            a.nseq = 2; a.max_draft = 3; a.vocab = 1000; a.ld_target = a.ld_draft = 1000;
            a.target_dev = a.accept_u_dev = a.sample_u_dev = (float*)ptr;
            a.draft_ids_dev = a.out_ids_dev = (uint32_t*)ptr;
            a.n_draft_dev = a.out_n_dev = (int32_t*)ptr;
            rc = laic::verify_drafts(0, a, nullptr, {pdl != 0, &n});
        }
        if (rc) return 1;
        std::printf("%d", n);
        for (int e : early) std::printf(" %d", e);
        std::printf("\n");
    }
    return 0;
}
