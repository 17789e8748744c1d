// lookup_buffers.h - which of a lookup call's results may lie over what it reads (host only, no device code).
//
// Workgroups of one launch read az, ax and the vectors while others store results, so a result may not touch memory that another
// instance or component is read from.  Exact identity is a different matter: a_new, v and n_eff of an instance are stored by the
// workgroup that has read the instance's scalars, and b_new of a component by the thread that has read its b_old.
#pragma once
#include <stddef.h>
#include <stdint.h>

struct LkBuffers {
    // read; null: not part of the call
    const void *az, *ax, *a_old, *bz, *bx, *b_old;
    // stored; null: not asked for
    const void *a_new, *v, *n_eff, *b_new, *r;
    size_t scal, nz, nx, nout;       // bytes of a scalar array, of bz, of bx, of b_old / b_new / r
};

static inline bool lk_overlap(const void* x, size_t nx, const void* y, size_t ny) {
    const uintptr_t a = (uintptr_t)x, b = (uintptr_t)y;
    return x && y && a < b + ny && b < a + nx;
}

// null, or why the call is refused
static inline const char* lk_conflict(const LkBuffers& m) {
    const struct { const void* p; size_t n; bool scalar; } in[] = {{m.az, m.scal, true}, {m.ax, m.scal, true}, {m.a_old, m.scal, true},
                                                                   {m.bz, m.nz, false}, {m.bx, m.nx, false}, {m.b_old, m.nout, false}},
                                                           out[] = {{m.a_new, m.scal, true}, {m.v, m.scal, true}, {m.n_eff, m.scal, true},
                                                                    {m.b_new, m.nout, false}, {m.r, m.nout, false}};
    for (int i = 0; i < 5; ++i)
        for (int j = 0; j < i; ++j)
            if (lk_overlap(out[i].p, out[i].n, out[j].p, out[j].n)) return "two results overlap";
    for (const auto& o : out)
        for (const auto& s : in) {
            const bool in_place = o.p == s.p && ((o.scalar && s.scalar) || (o.p == m.b_new && s.p == m.b_old && !s.scalar));
            if (!in_place && lk_overlap(o.p, o.n, s.p, s.n)) return "a result overlaps what the call reads";
        }
    return nullptr;
}

// does a scalar result replace a precision that every workgroup of the instance reads?
static inline bool lk_scalars_in_place(const void* az, const void* ax, const void* a_new, const void* v, const void* n_eff) {
    for (const void* o : {a_new, v, n_eff})
        if (o && (o == az || o == ax)) return true;
    return false;
}
