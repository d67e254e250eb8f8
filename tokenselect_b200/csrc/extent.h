// Whether what one pointer of a call covers meets what another covers; host only.
#pragma once
#include <stdint.h>

namespace ts {

// `n` rows of `bytes`, `step` apart.
struct Extent {
    uintptr_t at;
    uint64_t bytes, step, n;
    Extent(const void* p, uint64_t row_bytes, uint64_t row_step = 0, uint64_t rows = 1)
        : at(reinterpret_cast<uintptr_t>(p)), bytes(row_bytes), step(row_step), n(p != nullptr && row_bytes > 0 ? rows : 0) {
        if (n > 1 && step <= bytes) { bytes += (n - 1) * step; n = 1; }       // without gaps
    }
    uintptr_t end() const { return at + (n - 1) * step + bytes; }
    // the rows meet [from, to)
    bool meets(uintptr_t from, uintptr_t to) const {
        if (n == 0 || from >= to || to <= at) return false;
        const uint64_t i = n == 1 || from < at + bytes ? 0 : (from - at - bytes) / step + 1;      // first row that ends behind `from`
        return i < n && at + i * step < to && from < at + i * step + bytes;
    }
};
inline bool overlap(const Extent& a, const Extent& b) {
    if (a.n == 0 || b.n == 0 || a.end() <= b.at || b.end() <= a.at) return false;
    if (a.n == 1) return b.meets(a.at, a.at + a.bytes);
    if (b.n == 1) return a.meets(b.at, b.at + b.bytes);
    // Slices of one buffer: their places repeat with the steps' greatest common divisor.
    uint64_t g = a.step, r = b.step;
    while (r != 0) { const uint64_t t = g % r; g = r; r = t; }
    const uint64_t off = b.at >= a.at ? (b.at - a.at) % g : (g - (a.at - b.at) % g) % g;
    if (off >= a.bytes && off + b.bytes <= g) return false;
    const Extent& few = a.n <= b.n ? a : b;
    const Extent& many = a.n <= b.n ? b : a;
    for (uint64_t i = 0; i < few.n; ++i)
        if (many.meets(few.at + i * few.step, few.at + i * few.step + few.bytes)) return true;
    return false;
}

}  // namespace ts
