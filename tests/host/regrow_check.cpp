// One growing buffer under an allocator that fails at a chosen call: per query "fail_at need..." on stdin, for each need
// the error, whether the buffer moved, whether there is one, and its capacity.
#include <cstdio>
#include <cstdlib>
#include <iostream>
#include <sstream>
#include <string>

#include "buffers.h"

int main() {
    std::string line;
    while (std::getline(std::cin, line)) {
        std::istringstream in(line);
        int fail_at = 0, calls = 0, live = 0;
        size_t need = 0, cap = 0;
        void* p = nullptr;
        in >> fail_at;
        while (in >> need) {
            bool moved = false;
            const int e = laic::regrow(&p, cap, need, 4, moved,
                                       [&](void** q, size_t bytes) {
                                           if (calls++ == fail_at) return 2;
                                           *q = std::malloc(bytes);
                                           ++live;
                                           return 0;
                                       },
                                       [&](void* q) { std::free(q); --live; });
            std::printf("%d:%d:%d:%zu ", e, moved ? 1 : 0, p ? 1 : 0, cap);
            if (live != (p ? 1 : 0)) return 1;
        }
        std::printf("\n");
        std::free(p);
    }
    return 0;
}
