// Launches of the serving operators (serving.cu), used by its entry points and by the engine.
#pragma once
#include <cuda_runtime.h>

#include <string>

#include "../../include/laic_b200.h"

#include "errors.h"

namespace laic {

// Records the calling thread's error message (laic_last_error) and returns `code` (engine.cu).
int api_fail(int code, const std::string& msg);

// How an operator's kernels are launched: whether the first may start while its predecessor in the stream drains
// (and each later one behind the one before it), and a count that its launches are added to.
struct LaunchOpts {
    bool pdl = true;
    int* launches = nullptr;
};

// The checks and launches behind the entry points of the same names.
int kv_append(const laic_kv_pages& pages, const laic_kv_append_args& a, cudaStream_t st, LaunchOpts o = {});
int kv_attention_bytes(const laic_kv_pages& pages, const laic_kv_attention_args& a, uint64_t* bytes);
int kv_attention(const laic_kv_pages& pages, const laic_kv_attention_args& a, cudaStream_t st, LaunchOpts o = {});
int logits_probs(int device, int rows, int vocab, const float* x, long long ldx, const float* temp, float* y, long long ldy,
                 cudaStream_t st, LaunchOpts o = {});
int verify_drafts(int device, const laic_verify_args& a, cudaStream_t st, LaunchOpts o = {});
// Kernel attributes (call before any graph capture; the entry points call it themselves).
cudaError_t serving_set_attributes();

}  // namespace laic
