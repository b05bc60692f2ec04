// Sets of buffers under an allocator that fails at a chosen call: prints, per query "buffers fail_at" on stdin, for
// each attempt until one succeeds: the error, the allocations made in it, the buffers present.
#include <cstdio>
#include <cstdlib>
#include <iostream>
#include <vector>

#include "buffers.h"

int main() {
    int n = 0, fail_at = 0;
    while (std::cin >> n >> fail_at) {
        void* b[3] = {nullptr, nullptr, nullptr};
        int calls = 0, made = 0;
        auto alloc = [&](void** p, size_t bytes) {
            if (calls++ == fail_at) return 2;
            *p = std::malloc(bytes);
            ++made;
            return 0;
        };
        for (int e = 1; e;) {
            made = 0;
            e = laic::alloc_missing({{&b[0], 8}, {&b[1], n > 1 ? size_t(16) : 0}, {&b[2], n > 2 ? size_t(4) : 0}}, alloc);
            std::printf("%d:%d:%d ", e, made, (b[0] != nullptr) + (b[1] != nullptr) + (b[2] != nullptr));
        }
        std::printf("\n");
        for (void* p : b) std::free(p);
    }
    return 0;
}
