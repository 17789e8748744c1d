// workspace.h - growth of a context's workspace (host only, no device code).
#pragma once
#include <stddef.h>

#include <initializer_list>

constexpr size_t kWsFirst = (size_t)4 << 20;     // a new context's

// The size to ask for when `have` does not hold `need`: doubled, so that a caller whose needs grow step by step does not
// re-allocate at every step.
static inline size_t ws_next(size_t have, size_t need) {
    size_t n = have > kWsFirst ? have : kWsFirst;
    while (n < need) {
        if (n > (size_t)-1 / 2) return need;
        n *= 2;
    }
    return n;
}

// Replaces the workspace by one of at least `need` bytes.  alloc(bytes): a new one or null.  If the doubled size is not to be had,
// exactly the need is tried; if that is not to be had either, the old size comes back, so that smaller calls go on.  False: the
// workspace does not hold `need` (`*ws` and `*have` say what there is, at worst null and 0).
template <typename Alloc, typename Free> static bool ws_grow(void** ws, size_t* have, size_t need, Alloc alloc, Free release) {
    const size_t old = *have;
    if (*ws) release(*ws);
    *ws = nullptr;
    *have = 0;
    for (const size_t n : {ws_next(old, need), need, old > kWsFirst ? old : kWsFirst}) {
        *ws = alloc(n);
        if (*ws) {
            *have = n;
            break;
        }
    }
    return *ws && *have >= need;
}
