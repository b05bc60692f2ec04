// Host-side check of the page table row a group is read through (paged_attn.cuh): a query per line,
//   r0 r1 rows nseq hasseq len... seq...   -> sequence err
#include <cstdio>
#include <iostream>
#include <sstream>
#include <string>
#include <vector>

#include "paged_attn.cuh"

int main() {
    std::string line;
    while (std::getline(std::cin, line)) {
        std::istringstream in(line);
        auto ints = [&](int n) {
            std::vector<int> v(n);
            for (int& x : v) in >> x;
            return v;
        };
        auto a = ints(5);
        auto len = ints(a[2]);
        std::vector<int> seq = a[4] ? ints(a[2]) : std::vector<int>();
        int err = 0;
        laic::KvAttnParams p{};
        p.err = &err;
        p.rows = a[2]; p.nseq = a[3]; p.len = len.data(); p.seq = a[4] ? seq.data() : nullptr;
        const int s = laic::group_seq(p, a[0], a[1], laic::row_at(p, a[0]));
        std::printf("%d %d\n", s, err);
    }
    return 0;
}
