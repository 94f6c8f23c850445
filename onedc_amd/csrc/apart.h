// apart.h — do two operands of a call lie in the same memory?  (host side, before a launch)
#pragma once
#include <cstdint>
#include <numeric>

struct OnedcMem {
    uintptr_t lo = 0, hi = 0;             // first byte and end; nothing: equal
    int64_t pitch = 0, width = 0;         // bytes between the beginnings of its rows (0: one row), bytes of a row
};
inline OnedcMem onedc_mem(const void *p, int64_t bytes) {
    if (!p || bytes <= 0) return {};
    return {(uintptr_t)p, (uintptr_t)p + bytes, 0, bytes};
}
// rows of `channels` values of `size` bytes, `cs` values apart, from value `co` on
inline OnedcMem onedc_mem_rows(const void *p, int64_t rows, int64_t cs, int64_t co, int64_t channels, int size) {
    if (!p || rows <= 0) return {};
    const uintptr_t lo = (uintptr_t)p + co * size;
    return {lo, lo + ((rows - 1) * cs + channels) * size, rows > 1 ? cs * size : 0, channels * size};
}
// false: no byte is in both.  Operands whose ranges meet are still apart where they are other columns of a common grid of rows.
inline bool onedc_mem_shared(const OnedcMem &a, const OnedcMem &b) {
    if (a.lo == a.hi || b.lo == b.hi || a.hi <= b.lo || b.hi <= a.lo) return false;
    const int64_t grid = std::gcd(a.pitch, b.pitch);
    if (!grid) return true;
    const int64_t d = (int64_t)(b.lo - a.lo) % grid, at = d < 0 ? d + grid : d;
    return at < a.width || at + b.width > grid;
}
template <int N, int M>
inline bool onedc_mem_any_shared(const OnedcMem (&outs)[N], const OnedcMem (&others)[M]) {
    for (const OnedcMem &o : outs)
        for (const OnedcMem &m : others)
            if (onedc_mem_shared(o, m)) return true;
    return false;
}
