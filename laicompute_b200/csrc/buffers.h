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

}  // namespace laic
