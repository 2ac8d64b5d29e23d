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
// (tokens, heads, dim) from its lowest element to its highest.
inline Stretch rows_at(const void* p, int64_t tokens, int64_t heads, int64_t token, int64_t head, int64_t dim) {
    const int64_t t = (tokens - 1) * token, h = (heads - 1) * head;
    const uintptr_t x = reinterpret_cast<uintptr_t>(p);
    return {x + 2 * ((t < 0 ? t : 0) + (h < 0 ? h : 0)), x + 2 * ((t > 0 ? t : 0) + (h > 0 ? h : 0) + dim)};
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
    // Pages that are equally far apart may lie between one another; of other pairs the whole stretches are compared.
    bool meets(const Pages& o) const {
        const Stretch mine = elements_at(at, (count - 1) * stride + elements), theirs = elements_at(o.at, (o.count - 1) * o.stride + o.elements);
        if (!mine.meets(theirs)) return false;
        if (count == 1) return o.meets(mine);
        if (o.count == 1) return meets(theirs);
        if (stride != o.stride) return true;
        // page i of these and j of those: only those with i - j next to (o.at - at) / stride can meet
        const uintptr_t x = mine.from, y = theirs.from;
        const int64_t apart = x < y ? (int64_t)((y - x) / (2 * stride)) : -(int64_t)((x - y) / (2 * stride));
        for (int64_t m = apart - 1; m <= apart + 1; ++m) {
            if (m >= count || -m >= o.count) continue;
            const uintptr_t shifted = x + 2 * m * stride;      // page m + j of these against page j of those
            if (Stretch{shifted, shifted + 2 * elements}.meets({y, y + 2 * o.elements})) return true;
        }
        return false;
    }
};

}  // namespace hqm
