// Host-side checks of the paged cache's index rules (paged.cuh, paged_attn.cuh): reads one query per
// line from stdin and prints what the kernels would use.
//   place seq pos nseq pps shift npages positions table...      -> page bad
//   row r rows nseq pps shift max_len shared hasseq len... seq... -> n shared seq err
//   group g rows groups nseq pps shift max_rows max_shared start... len... -> ok r0 r1 shared err
#include <climits>
#include <cstdio>
#include <iostream>
#include <sstream>
#include <string>
#include <vector>

#include "paged_attn.cuh"

int main() {
    std::string line, what;
    while (std::getline(std::cin, line)) {
        std::istringstream in(line);
        in >> what;
        auto ints = [&](int n) {
            std::vector<int> v(n);
            for (int& x : v) in >> x;
            return v;
        };
        int err = 0;
        laic::KvAttnParams p{};
        p.err = &err;
        if (what == "place") {
            auto a = ints(7);
            auto table = ints(a[2] * a[3]);
            int bad = 0;
            const int page = laic::kv_place(a[0], a[1], table.data(), a[2], a[3], a[4], a[5], a[6], bad);
            std::printf("%d %d\n", page, bad);
        } else if (what == "row") {
            auto a = ints(8);
            auto len = ints(a[1]);
            std::vector<int> seq = a[7] ? ints(a[1]) : std::vector<int>();
            p.rows = a[1]; p.nseq = a[2]; p.pages_per_seq = a[3]; p.page_shift = a[4]; p.max_len = a[5];
            p.len = len.data(); p.seq = a[7] ? seq.data() : nullptr;
            const laic::RowView v = laic::row_view(p, a[0], a[6]);
            std::printf("%d %d %d %d\n", v.n, v.shared, v.seq, err);
        } else {
            auto a = ints(8);
            auto start = ints(a[2] + 1);
            auto len = ints(a[2]);
            p.rows = a[1]; p.groups = a[2]; p.nseq = a[3]; p.pages_per_seq = a[4]; p.page_shift = a[5];
            p.max_group_rows = a[6]; p.max_shared = a[7];
            p.group_rows = start.data(); p.group_len = len.data();
            int r0 = 0, r1 = 0;
            const bool ok = laic::group_rows(p, a[0], r0, r1);
            const int sh = ok && r1 > r0 ? laic::group_shared(p, a[0]) : 0;
            std::printf("%d %d %d %d %d\n", ok ? 1 : 0, r0, r1, sh, err);
        }
    }
    return 0;
}
