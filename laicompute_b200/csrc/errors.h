// What kernels leave in an engine's error words, and the messages the host makes of them (plain C++).
#pragma once
#include <string>

namespace laic {

// Codes a bounded device wait writes into its launch's error word when it runs
// out (about one second of SM clocks); the host turns them into messages.
enum : int {
    kErrMbarrier = 1,     // a bulk copy into shared memory never completed (mbarrier wait)
    kErrTeamMerge = 2,    // a warp team's partial-sum slot was never released
    kErrGridBarrier = 3,  // a persistent kernel's grid barrier was not reached by every CTA
    kErrPeerFlag = 4,     // a tensor-parallel peer never published its allreduce slice
    kErrDepCounter = 5,   // a persistent kernel's dependency counter never reached its target
};

// Bits of a paged cache's error word (LAIC_KV_* of the public header): another word than that of the codes above,
// whose values they share.
enum : int { kKvBadSeq = 1, kKvBadPos = 2, kKvBadPage = 4, kKvBadGroup = 8, kKvWait = 16 };

inline std::string wait_error_text(int code) {
    switch (code) {
    case kErrMbarrier: return "device wait timed out: a bulk copy into shared memory never completed";
    case kErrTeamMerge: return "device wait timed out: a matvec warp team's partial-sum slot was never released";
    case kErrGridBarrier: return "device wait timed out: a decode-step grid barrier was not reached by every CTA";
    case kErrPeerFlag: return "device wait timed out: a tensor-parallel peer never published its allreduce slice";
    case kErrDepCounter: return "device wait timed out: a decode-step dependency counter never reached its target";
    }
    return "device wait timed out (code " + std::to_string(code) + ")";
}

inline std::string kv_error_text(int bits) {
    std::string s = "paged KV cache:";
    if (bits & kKvBadSeq) s += " sequence index outside the page table;";
    if (bits & kKvBadPos) s += " position or length beyond its bound;";
    if (bits & kKvBadPage) s += " page id out of range;";
    if (bits & kKvBadGroup) s += " group rows out of order or above their bound;";
    if (bits & kKvWait) s += " a device wait timed out;";
    s.pop_back();
    return s;
}

// A step's two words together: "" where both are zero.
inline std::string step_error_text(int wait_code, int kv_bits) {
    std::string s = wait_code ? wait_error_text(wait_code) : "";
    if (kv_bits) s += (s.empty() ? "" : "; ") + kv_error_text(kv_bits);
    return s;
}

}  // namespace laic
