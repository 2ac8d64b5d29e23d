// Whether what a kernel writes shares memory with what it reads: its CTAs run in any order, so one may have written what another has
// yet to read.  Elements of two bytes, strides in elements.
#pragma once
#include <stdint.h>

namespace hqm {

struct Stretch {                 // bytes from .. to - 1
    uintptr_t from, to;
    bool meets(const Stretch& o) const { return from < o.to && o.from < to; }
};
inline Stretch elements_at(const void* p, int64_t n) {
    const uintptr_t x = reinterpret_cast<uintptr_t>(p);
    return {x, x + 2 * n};
}
// (tokens, heads, dim) from its first element to its last.
inline Stretch rows_at(const void* p, int64_t tokens, int64_t heads, int64_t token, int64_t head, int64_t dim) {
    return elements_at(p, (tokens - 1) * token + (heads - 1) * head + dim);
}

// `count` pages of `elements` each, `stride` >= elements apart: what lies between them is not theirs.
struct Pages {
    const void* at;
    int64_t count, stride, elements;
    bool meets(const Stretch& s) const {
        const uintptr_t x = reinterpret_cast<uintptr_t>(at);
        if (s.to <= x || s.from >= s.to) return false;
        // the first page that ends behind s.from
        const int64_t i = s.from < x + 2 * elements ? 0 : (int64_t)((s.from - x - 2 * elements) / (2 * stride)) + 1;
        return i < count && x + 2 * i * stride < s.to;
    }
};

}  // namespace hqm
