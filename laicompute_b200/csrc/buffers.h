// Sets of device buffers that stay consistent where an allocation fails (plain C++: the allocator is the caller's).
#pragma once
#include <cstddef>
#include <initializer_list>

namespace laic {

struct Want {
    void** at;
    size_t bytes;
};
// Makes the buffers of `set` that are missing (null) with alloc(void**, bytes), which returns 0 or its error; the
// first error is returned. What was made stays, and the next call makes the rest.
template <typename Alloc>
auto alloc_missing(std::initializer_list<Want> set, Alloc&& alloc) -> decltype(alloc((void**)nullptr, (size_t)0)) {
    for (const Want& w : set)
        if (!*w.at && w.bytes) {
            void* p = nullptr;
            if (auto e = alloc(&p, w.bytes)) return e;
            *w.at = p;
        }
    return {};
}

// Replaces *p, which holds `cap` elements of `size` bytes, where `need` is above that. `moved` is set as soon as the old
// buffer is gone; where the new one fails there is none, and `cap` is zero.
template <typename Alloc, typename Free>
auto regrow(void** p, size_t& cap, size_t need, size_t size, bool& moved, Alloc&& alloc, Free&& release)
    -> decltype(alloc((void**)nullptr, (size_t)0)) {
    if (need <= cap) return {};
    if (*p) release(*p);
    *p = nullptr;
    cap = 0;
    moved = true;
    if (auto e = alloc(p, need * size)) {
        *p = nullptr;
        return e;
    }
    cap = need;
    return {};
}

}  // namespace laic
