"""GPU: norms over lists of arrays, clipping, bounded steps, and iterate(max_step=...).

The kernels sum squares in double: n terms are off by at most (n + 2) 2^-53 relative (all terms are positive), half of that
after the root, on either side.  A clipped value is off by the factor's error plus one rounding to the element type."""
import ctypes as C

import numpy as np
import pytest

from oracle import tramp_oracle as orc
from tests.lookup_plain import LookupFactor, clip_plain, step_plain, zipf_tokens

pytestmark = pytest.mark.gpu
U = 2.0**-53

LISTS = [(1,), (3,), (4097,), (1, 1, 1), (0, 5, 0), (4096, 8192), (17, 4095, 4096, 4097, 3), (100003,), (5, 300001, 2, 70000), tuple(range(1, 90)),
         (5000011,)]


def arrays_of(rs, lengths, batch, dtype, scale=1.0):
    return [(scale * rs.standard_normal((batch, n))).astype(dtype) for n in lengths]


def group(T, ctx, arrays, dtype):
    return T.ArrayGroup([ctx.array(a, dtype) for a in arrays])


def get(g):
    return [a.get() for a in g.arrays]


@pytest.mark.parametrize("dtype", [np.float64, np.float32])
@pytest.mark.parametrize("batch", [1, 3])
@pytest.mark.parametrize("lengths", LISTS, ids=lambda s: f"{len(s)}x{max(s)}")
def test_norm_clip_step(ctx, lengths, batch, dtype):
    import tramp_amd as T
    rs = np.random.RandomState(sum(lengths) + batch)
    x, p = arrays_of(rs, lengths, batch, dtype), arrays_of(rs, lengths, batch, dtype)
    n = sum(lengths)
    rel = 2 * (n + 4) * U
    half = np.finfo(dtype).eps / 2
    norm0, _ = clip_plain(x, 1.0)
    g, gp, out = group(T, ctx, x, dtype), group(T, ctx, p, dtype), group(T, ctx, p, dtype)
    got = g.norm().get()
    assert (np.abs(got - norm0) <= rel * norm0).all()
    for bound in (0.5 * norm0.max(), 1.001 * norm0.min(), 1e3 * norm0.max() + 1):     # all, some, none clipped
        _, want = clip_plain(x, bound)
        nn = g.clip(bound, out=out).get()
        assert np.array_equal(nn, got)
        for y, w, src in zip(get(out), want, x):
            assert (np.abs(y - w) <= (half + rel + 4 * U) * np.abs(w)).all()
            for b in range(batch):
                if nn[b] <= bound:
                    assert np.array_equal(y[b], src[b])
        assert all(np.array_equal(a, b) for a, b in zip(get(g), x))                   # the source is untouched
        ns, ws, c = step_plain(x, p, bound)
        nn = g.limit_step(gp, bound, out=out).get()
        assert (np.abs(nn - ns) <= rel * ns).all()
        for y, w, a, q in zip(get(out), ws, x, p):
            mag = np.abs(q.astype(float)) + np.abs(a.astype(float))
            assert (np.abs(y - w) <= half * np.abs(w) + (rel + 6 * U) * mag).all()
        assert all(np.array_equal(a, b) for a, b in zip(get(g), x)) and all(np.array_equal(a, b) for a, b in zip(get(gp), p))
    # in place, with precisions, and the refreshed copy
    bound = 0.5 * norm0.max()
    first = g.limit_step(gp, bound, out=out).get()
    kept = get(out)
    a, a0 = rs.uniform(1, 2, (5, batch)), rs.uniform(1, 2, (5, batch))
    ad, a0d = ctx.array(a), ctx.array(a0)
    nn = g.limit_step(gp, bound, a=ad, a_prev=a0d, refresh=True).get()
    assert np.array_equal(nn, first)
    c = np.where(nn > bound, bound / np.where(nn > 0, nn, 1), 1.0)
    want = np.where(c < 1, a0 + c * (a - a0), a)
    assert (np.abs(ad.get() - want) <= 8 * U * (np.abs(a) + np.abs(a0))).all() and np.array_equal(ad.get(), a0d.get())
    for y, w, q in zip(get(g), kept, get(gp)):
        assert np.array_equal(y, w) and np.array_equal(y, q)


@pytest.mark.parametrize("dtype", [np.float64, np.float32])
def test_norms_that_are_not_finite(ctx, dtype):
    import tramp_amd as T
    x = [np.array([[1, 2], [np.nan, 1], [np.inf, 1], [0, 0]], dtype), np.array([[2], [1], [1], [0]], dtype)]
    p = [np.zeros((4, 2), dtype), np.zeros((4, 1), dtype)]
    g, gp = group(T, ctx, x, dtype), group(T, ctx, p, dtype)
    a, a0 = ctx.array(np.full((2, 4), 3.0)), ctx.array(np.full((2, 4), 1.0))
    n = g.limit_step(gp, 1.5, out=group(T, ctx, p, dtype), a=a, a_prev=a0).get()
    assert n[0] == 3.0 and np.isnan(n[1]) and n[2] == np.inf and n[3] == 0
    assert np.array_equal(a.get(), [[2, 3, 3, 3]] * 2)
    n = g.clip(1.5).get()
    assert n[0] == 3.0 and np.isnan(n[1]) and n[2] == np.inf and n[3] == 0
    y = get(g)
    assert np.array_equal(y[0][0], np.array([0.5, 1.0], dtype)) and y[1][0, 0] == 1.0
    for b in (1, 2, 3):
        assert np.array_equal(y[0][b], x[0][b], equal_nan=True) and np.array_equal(y[1][b], x[1][b])
    # squares beyond the element type's range
    big = np.full((1, 3), 1e30, dtype)
    g = group(T, ctx, [big], dtype)
    assert g.clip(1.0).get()[0] == pytest.approx(np.sqrt(3) * float(big[0, 0]), rel=1e-12)
    assert get(g)[0] == pytest.approx(np.full((1, 3), 1 / np.sqrt(3)), rel=1e-6)
    assert np.array_equal(group(T, ctx, x, dtype).clip(np.inf).get(), n, equal_nan=True)


@pytest.mark.parametrize("dtype", [np.float64, np.float32])
def test_views_at_any_boundary_and_nothing_behind(ctx, dtype):
    import tramp_amd as T
    rs = np.random.RandomState(1)
    item = np.dtype(dtype).itemsize
    data = [rs.standard_normal((2, n)).astype(dtype) for n in (5, 4099, 64)]
    want = None
    for shift in range(4):
        keep = [ctx.array(np.concatenate([np.full(shift, 7, dtype), d.ravel(), np.full(5, 7, dtype)]), dtype) for d in data]
        other = [ctx.array(np.concatenate([np.full(3 - shift, 7, dtype), 0 * d.ravel(), np.full(5, 7, dtype)]), dtype) for d in data]
        g = T.ArrayGroup([T.DeviceArray(ctx, d.shape, dtype, ptr=k.ptr + shift * item, owner=False) for d, k in zip(data, keep)])
        o = T.ArrayGroup([T.DeviceArray(ctx, d.shape, dtype, ptr=k.ptr + (3 - shift) * item, owner=False) for d, k in zip(data, other)])
        res = [g.clip(3.0, out=o).get()] + get(o)
        g.limit_step(o, 1.0)
        res += get(g)
        for k, s in [(k, shift) for k in keep] + [(k, 3 - shift) for k in other]:
            h = k.get()
            assert (h[:s] == 7).all() and (h[-5:] == 7).all()
        want = want or res
        assert all(np.array_equal(a, b) for a, b in zip(res, want))


@pytest.mark.parametrize("dtype, batch, lengths, inplace", [(np.float64, 6, (1500001, 1000000), False), (np.float64, 6, (1500001, 1000000), True),
                                                            (np.float32, 1, (30000001, 5, 10000000), True), (np.float32, 37, (300007,), False)])
def test_large_lists(ctx, dtype, batch, lengths, inplace):
    "slices of instances, accesses past the caches: the same results, nothing but the arrays touched"
    import tramp_amd as T
    rs = np.random.RandomState(4)
    x = [rs.standard_normal((batch, n)).astype(dtype) * (1 + np.arange(batch)[:, None]) for n in lengths]
    p = [(0.5 * rs.standard_normal((batch, n))).astype(dtype) for n in lengths]
    x = [v.astype(dtype) for v in x]
    g, gp = group(T, ctx, x, dtype), group(T, ctx, p, dtype)
    out = g if inplace else group(T, ctx, p, dtype)
    norm, want, c = step_plain(x, p, 1.0)
    bound = float(np.median(norm)) * 0.9
    norm, want, c = step_plain(x, p, bound)
    got = g.limit_step(gp, bound, out=None if inplace else out).get()
    rel = 2 * (sum(lengths) + 4) * U
    assert (np.abs(got - norm) <= rel * norm).all()
    half = np.finfo(dtype).eps / 2
    for y, w, a, q in zip(get(out), want, x, p):
        mag = np.abs(q.astype(float)) + np.abs(a.astype(float))
        assert (np.abs(y - w) <= half * np.abs(w) + (rel + 6 * U) * mag).all()
    assert all(np.array_equal(a, b) for a, b in zip(get(gp), p))


def test_overlaps_are_refused(ctx):
    import tramp_amd as T
    a = ctx.array(np.arange(20.0))
    view = lambda lo, n: T.DeviceArray(ctx, (n,), np.float64, ptr=a.ptr + 8 * lo, owner=False)      # noqa: E731
    E = T._lib.TrampHipError
    with pytest.raises(E):
        T.ArrayGroup([view(0, 5), view(4, 5)])
    with pytest.raises(E):
        T.ArrayGroup([view(0, 5), view(0, 5)])
    g = T.ArrayGroup([view(0, 5), view(5, 5)])
    shifted, swapped, apart = T.ArrayGroup([view(1, 5), view(10, 5)]), T.ArrayGroup([view(5, 5), view(0, 5)]), T.ArrayGroup([view(10, 5), view(15, 5)])
    for bad in (shifted, swapped):
        with pytest.raises(E):
            g.clip(1.0, out=bad)
        with pytest.raises(E):
            g.limit_step(bad, 1.0)
        with pytest.raises(E):
            g.limit_step(apart, 1.0, out=bad)
    with pytest.raises(E):
        g.limit_step(g, 1.0)
    with pytest.raises(E):
        g.limit_step(apart, 1.0, out=apart)
    with pytest.raises(E):
        g.limit_step(apart, 1.0, a=a.reshape(20, 1), a_prev=a.reshape(20, 1))
    assert np.array_equal(a.get(), np.arange(20.0))
    g.limit_step(apart, 1e9)
    assert np.array_equal(a.get(), np.arange(20.0))


def test_norms_and_precisions_inside_a_list_are_refused(ctx):
    import tramp_amd as T
    E = T._lib.TrampHipError
    m = ctx.array(np.arange(40.0))
    view = lambda lo, *shape: T.DeviceArray(ctx, shape, np.float64, ptr=m.ptr + 8 * lo, owner=False)      # noqa: E731
    g, prev, out = (T.ArrayGroup([view(lo, 2, 2), view(lo + 4, 2, 3)]) for lo in (0, 10, 20))
    apart = T.ArrayGroup([view(0, 2, 2)])
    a, a_prev, norm = view(30, 1, 2), view(32, 1, 2), view(34, 2)
    for bad in (view(9, 2), view(0, 2), view(3, 2)):
        with pytest.raises(E):
            g.norm(bad)
        with pytest.raises(E):
            g.clip(1.0, norm=bad)
    with pytest.raises(E):
        g.clip(1.0, out=out, norm=view(28, 2))
    for kw in (dict(norm=view(9, 2)), dict(norm=view(10, 2)), dict(norm=view(29, 2)), dict(norm=view(31, 2)), dict(norm=view(33, 2)),
               dict(a=view(0, 1, 2)), dict(a=view(29, 1, 2)), dict(a_prev=view(18, 1, 2)), dict(a_prev=view(31, 1, 2))):
        with pytest.raises(E):
            g.limit_step(prev, 1.0, out=out, **dict(dict(norm=norm, a=a, a_prev=a_prev), **kw))
    apart.norm(view(4, 2))                                             # right behind the array
    assert np.array_equal(m.get()[np.r_[:4, 6:40]], np.arange(40.0)[np.r_[:4, 6:40]])
    g.limit_step(prev, 1.0, out=out, norm=norm, a=a, a_prev=a_prev)


def test_precisions_that_are_infinite_stay_so(ctx):
    import tramp_amd as T
    for n in (3, 50000):                                               # one launch, two launches
        x, p = T.ArrayGroup([ctx.array(np.full((1, n), 2.0))]), T.ArrayGroup([ctx.zeros((1, n), np.float64)])
        a, a_prev = ctx.array(np.array([[np.inf], [4.0], [np.inf]])), ctx.array(np.array([[np.inf], [2.0], [1.0]]))
        norm = x.limit_step(p, np.sqrt(n), a=a, a_prev=a_prev).get()   # factor 1/2
        assert norm[0] == pytest.approx(2 * np.sqrt(n), rel=1e-14)
        assert a.get()[:, 0] == pytest.approx([np.inf, 3.0, np.inf], rel=1e-14)


@pytest.mark.parametrize("n", [3, 50000])                              # one launch, two launches
@pytest.mark.parametrize("refresh", [False, True])
def test_precisions_whose_step_is_not_finite_take_it_whole(ctx, n, refresh):
    import tramp_amd as T
    x, p = T.ArrayGroup([ctx.array(np.full((1, n), 2.0))]), T.ArrayGroup([ctx.zeros((1, n), np.float64)])
    new, old = np.array([[4.0], [np.inf], [3.0], [np.nan], [-1e308], [5.0]]), np.array([[np.inf], [4.0], [np.nan], [2.0], [1e308], [1.0]])
    a, a_prev = ctx.array(new), ctx.array(old)
    norm = x.limit_step(p, np.sqrt(n), a=a, a_prev=a_prev, refresh=refresh).get()      # factor 1/2
    assert norm[0] == pytest.approx(2 * np.sqrt(n), rel=1e-14)
    assert np.array_equal(a.get()[:5], new[:5], equal_nan=True) and a.get()[5, 0] == pytest.approx(3.0, rel=1e-14)
    assert np.array_equal(a_prev.get(), a.get() if refresh else old, equal_nan=True)


def test_replays_equal_the_eager_calls(ctx):
    import tramp_amd as T
    rs = np.random.RandomState(9)
    x, p = arrays_of(rs, (300001, 77), 2, np.float32), arrays_of(rs, (300001, 77), 2, np.float32)
    y = arrays_of(rs, (10, 11), 5, np.float64)
    g, gp, o = (group(T, ctx, v, np.float32) for v in (x, p, p))
    h, ho = group(T, ctx, y, np.float64), group(T, ctx, y, np.float64)
    n1, n2 = ctx.empty((2,)), ctx.empty((5,))

    def first():
        g.limit_step(gp, 100.0, out=o, norm=n1)

    def second():
        h.clip(1.0, out=ho, norm=n2)
    first(), second()
    want = get(o) + [n1.get()] + get(ho) + [n2.get()]
    graphs = []
    for f in (first, second):
        ctx._call("tramp_graph_begin")
        f()
        gr = C.c_void_p()
        ctx._call("tramp_graph_end", C.byref(gr))
        graphs.append(gr)
    try:
        for _ in range(4):
            for t in o.arrays + ho.arrays + [n1, n2]:
                t.fill(0.0)
            for gr in graphs:
                ctx._call("tramp_graph_launch", gr)
            assert all(np.array_equal(a, b) for a, b in zip(get(o) + [n1.get()] + get(ho) + [n2.get()], want))
            g.norm()
            ctx.sync()
    finally:
        for gr in graphs:
            ctx._call("tramp_graph_destroy", gr)


# ---------------------------------------------------------------- iterate(max_step=...)
def ep_plain(factors, sizes, max_step, damping, iters):
    "the sweeps of orc.ep_chain, every message of an iteration then moved by min(1, max_step / |step|)"
    L = len(sizes)
    m = {(i, d): (0.0, np.zeros(sizes[i])) for i in range(L) for d in "fb"}
    damp = lambda o, n: tuple(damping * u + (1 - damping) * w for u, w in zip(o, n))       # noqa: E731
    norms = []
    for _ in range(iters):
        old = dict(m)
        for i in range(L):
            f = factors[i]
            new = f.forward(None, None, *m[i, "b"]) if i == 0 else f.forward(*m[i - 1, "f"], *m[i, "b"])
            m[i, "f"] = damp(old[i, "f"], new)
        for i in reversed(range(L)):
            f = factors[i + 1]
            new = f.backward(*m[i, "f"], None, None) if i == L - 1 else f.backward(*m[i, "f"], *m[i + 1, "b"])
            m[i, "b"] = damp(old[i, "b"], new)
        norm = np.sqrt(sum(np.sum((m[k][1] - old[k][1])**2) for k in m))
        norms.append(norm)
        c = min(1.0, max_step / norm) if norm > 0 else 1.0
        m = {k: tuple(o + c * (n - o) for o, n in zip(old[k], m[k])) for k in m}
    r = [(m[i, "f"][1] + m[i, "b"][1]) / (m[i, "f"][0] + m[i, "b"][0]) for i in range(L)]
    return r, norms


def problem(T, ctx, kind, B=3):
    rs = np.random.RandomState(7)
    V, n = 80, 300
    tok = zipf_tokens(rs, V, n, 1.0, 0.05)
    X = np.stack([orc.gb_sample(rs, V, 0.5) for _ in range(B)])
    if kind == "lookup":
        ch, ref = (lambda: T.LookupChannel(tok, V, padding_index=-1, ctx=ctx)), LookupFactor(tok, V)
        Z = np.stack([ref.lookup(x).reshape(-1) for x in X])
    else:
        n = 50
        W = orc.gaussian_ensemble(rs, n, V)
        ch, ref = (lambda: T.LinearChannel(W, ctx=ctx, svd="host")), orc.LinearFactor(W)
        Z = X @ W.T
    Y = Z + np.sqrt(0.1) * rs.standard_normal((B, n))
    lik = (lambda: T.GaussianLikelihood(y=Y, var=0.1, ctx=ctx)) if kind != "sgn" else (lambda: T.SgnLikelihood(y=np.where(Y > 0, 1.0, -1.0), ctx=ctx))
    make = lambda: T.ExpectationPropagation((T.GaussBernoulliPrior(size=V, rho=0.5, ctx=ctx) @ T.SISOVariable(id="x") @ ch()       # noqa: E731
                                             @ T.SISOVariable(id="z") @ lik()).to_model(), ctx=ctx)
    end = lambda b: orc.GaussLikFactor(Y[b], 0.1) if kind != "sgn" else orc.SgnLikFactor(np.where(Y[b] > 0, 1.0, -1.0))           # noqa: E731
    return make, [lambda b: [orc.GBPriorFactor(V, rho=0.5), ref, end(b)]][0], [V, n], X


@pytest.mark.parametrize("kind", ["lookup", "linear", "sgn"])
@pytest.mark.parametrize("damping", [0.0, 0.2])
@pytest.mark.parametrize("max_step", [3.0, 25.0])
def test_bounded_sweeps_match_the_plain_loop(ctx, kind, damping, max_step):
    import tramp_amd as T
    make, factors, sizes, _ = problem(T, ctx, kind)
    ep = make().iterate(max_iter=12, callback=T.PassCallback(), damping=damping or None, max_step=max_step)
    r, norms = ep.get_variables_data(), ep.step_norm.get()
    for b in range(3):
        want, nn = ep_plain(factors(b), sizes, max_step, damping, 12)
        for i, name in enumerate(("x", "z")):
            assert np.abs(r[name]["r"][b] - want[i]).max() < 1e-8 * np.abs(want[i]).max(), (name, b)
        assert norms[b] == pytest.approx(nn[-1], rel=1e-6)
    graph = make().iterate(max_iter=12, callback=T.PassCallback(), damping=damping or None, max_step=max_step, graph=True)
    kept = make().iterate(max_iter=12, callback=T.EarlyStoppingEP(tol=0.0, max_increase=np.inf), damping=damping or None, max_step=max_step,
                          restore_messages=True)
    kept_graph = make().iterate(max_iter=12, callback=T.EarlyStoppingEP(tol=0.0, max_increase=np.inf), damping=damping or None, max_step=max_step,
                                restore_messages=True, graph=True)
    for other in (graph, kept, kept_graph):
        for name in ("x", "z"):
            assert np.array_equal(other.get_variables_data()[name]["r"], r[name]["r"]), name


def conv_problem(T, ctx, depth):
    "a convolution (depth 1), or a dense layer and a convolution (depth 2): channels that keep projections of messages"
    rs = np.random.RandomState(21)
    n, B = 64, 2
    filt = rs.standard_normal(n) / 8
    W = np.stack([np.roll(filt, i) for i in range(n)])                    # x_i = sum_j f[j - i] z_j, roll(f, i)[j] = f[j - i]
    W0 = orc.gaussian_ensemble(rs, n, 40)
    Y = rs.standard_normal((B, n))
    conv, z = T.ConvChannel(filt, ctx=ctx), T.SISOVariable(id="z")
    assert np.abs(conv.sample(np.eye(n)).T - W).max() < 1e-13
    end = conv @ T.SISOVariable(id="c") @ T.GaussianLikelihood(y=Y, var=0.3, ctx=ctx)
    fac = lambda b: [orc.LinearFactor(W), orc.GaussLikFactor(Y[b], 0.3)]               # noqa: E731
    if depth == 1:
        model = T.GaussBernoulliPrior(size=n, rho=0.5, ctx=ctx) @ z @ end
        return model.to_model(), lambda b: [orc.GBPriorFactor(n, rho=0.5)] + fac(b), [n, n], ("z", "c")
    model = (T.GaussBernoulliPrior(size=40, rho=0.5, ctx=ctx) @ T.SISOVariable(id="x") @ T.LinearChannel(W0, ctx=ctx, svd="host") @ z @ end)
    return model.to_model(), lambda b: [orc.GBPriorFactor(40, rho=0.5), orc.LinearFactor(W0)] + fac(b), [40, n, n], ("x", "z", "c")


@pytest.mark.parametrize("graph", [False, True])
@pytest.mark.parametrize("restore", [False, True])
@pytest.mark.parametrize("depth", [1, 2])
def test_bounded_sweeps_over_channels_that_cache_projections(ctx, depth, restore, graph):
    import tramp_amd as T
    model, factors, sizes, names = conv_problem(T, ctx, depth)
    ep = T.ExpectationPropagation(model, ctx=ctx)
    ep.iterate(max_iter=9, callback=T.EarlyStoppingEP(tol=0.0, max_increase=np.inf), damping=0.1, max_step=4.0, restore_messages=restore, graph=graph)
    r, norms = ep.get_variables_data(), ep.step_norm.get()
    for b in range(2):
        want, nn = ep_plain(factors(b), sizes, 4.0, 0.1, 9)
        assert nn[0] > 4.0                                             # the bound is at work
        for i, name in enumerate(names):
            assert np.abs(r[name]["r"][b] - want[i]).max() < 1e-8 * np.abs(want[i]).max(), (name, b)
        assert norms[b] == pytest.approx(nn[-1], rel=1e-6)


def test_a_wide_bound_changes_nothing_and_bounds_end_with_their_call(ctx):
    import tramp_amd as T
    make, _, _, _ = problem(T, ctx, "lookup")
    free = make().iterate(max_iter=15, callback=T.PassCallback(), damping=0.1).get_variables_data()["x"]["r"]
    wide = make().iterate(max_iter=15, callback=T.PassCallback(), damping=0.1, max_step=1e12).get_variables_data()["x"]["r"]
    assert np.abs(free - wide).max() <= 1e-12 * np.abs(free).max()
    # a warm start without the bound goes on from the bounded messages, and a second bounded run starts anew
    ep = make()
    ep.iterate(max_iter=5, callback=T.PassCallback(), max_step=2.0)
    ep.iterate(max_iter=200, damping=0.3, warm_start=True)
    ref = make().iterate(max_iter=200, damping=0.3)
    assert (ep.status == 1).all() and np.abs(ep.get_variables_data()["x"]["r"] - ref.get_variables_data()["x"]["r"]).max() < 1e-3
    one = ep.iterate(max_iter=5, callback=T.PassCallback(), max_step=2.0).get_variables_data()["x"]["r"]
    two = make().iterate(max_iter=5, callback=T.PassCallback(), max_step=2.0).get_variables_data()["x"]["r"]
    assert np.array_equal(one, two)


def tree_model(T, ctx, tok, V, y, g):
    return (T.GaussianPrior(size=V, ctx=ctx) @ T.SIMOVariable(id="x", n_next=2) @ (
        (T.LookupChannel(tok, V, ctx=ctx) @ T.SISOVariable(id="z") @ T.GaussianLikelihood(y=y, var=0.2, ctx=ctx))
        + T.GaussianLikelihood(y=g, var=0.5, ctx=ctx))).to_model()


@pytest.mark.parametrize("restore", [False, True])
def test_on_a_tree(ctx, restore):
    "the table observed through a lookup and directly: exact posterior at the fixed point, reached with bounded sweeps too"
    import tramp_amd as T
    rs = np.random.RandomState(12)
    V, n = 25, 120
    tok = rs.randint(0, V, n)
    x = rs.standard_normal(V)
    y, g = x[tok] + 0.4 * rs.standard_normal(n), x + 0.7 * rs.standard_normal(V)
    count = np.bincount(tok, minlength=V)
    want = (np.bincount(tok, weights=y, minlength=V) / 0.2 + g / 0.5) / (1 + count / 0.2 + 1 / 0.5)
    kw = dict(max_iter=400, restore_messages=restore, callback=T.EarlyStoppingEP(tol=1e-10, max_increase=np.inf))
    steps = []
    for extra in (dict(), dict(max_step=5.0), dict(max_step=5.0, graph=True)):
        ep = T.ExpectationPropagation(tree_model(T, ctx, tok, V, y, g), ctx=ctx)
        ep.iterate(**kw, **extra)
        assert np.abs(ep.get_variables_data()["x"]["r"].reshape(-1) - want).max() < 1e-6
        steps.append(ep.n_iter)
    assert steps[1] == steps[2] > steps[0]


def test_a_step_that_is_not_finite_reaches_the_guard(ctx):
    import tramp_amd as T
    tok = np.zeros(4, int)
    y = np.array([[1.0, 2.0, 3.0, 4.0], [1.0, np.nan, 3.0, 4.0]])
    ep = T.ExpectationPropagation((T.GaussBernoulliPrior(size=2, rho=0.5, ctx=ctx) @ T.SISOVariable(id="x") @ T.LookupChannel(tok, 2, ctx=ctx)
                                   @ T.SISOVariable(id="z") @ T.GaussianLikelihood(y=y, var=0.1, ctx=ctx)).to_model(), ctx=ctx)
    with pytest.raises(ValueError, match="nan"):
        ep.iterate(max_iter=5, max_step=1.0)


@pytest.mark.parametrize("seed", range(3))
def test_uneven_counts_damped_and_bounded(ctx, seed):
    """A categorical regression that undamped sweeps do not solve: constant damping and a bounded step both meet the stopping rule, at
    one fixed point.  A run whose change falls below 1e-6 in at most 200 sweeps contracts by 1e-6 ** (1 / 200) = 0.933 a sweep or
    better, so it is within 1e-6 / (1 - 0.933) = 1.5e-5 of its fixed point; 1e-4 holds two of them."""
    import tramp_amd as T
    rs = np.random.RandomState(seed)
    V, n = 1000, 2000
    tok = zipf_tokens(rs, V, n, 1.0)
    x = orc.gb_sample(rs, V, 0.5)
    y = x[tok] + np.sqrt(0.1) * rs.standard_normal(n)
    r, sweeps = [], []
    for kw in (dict(damping=0.3), dict(max_step=10.0)):
        model = (T.GaussBernoulliPrior(size=V, rho=0.5, ctx=ctx) @ T.SISOVariable(id="x") @ T.LookupChannel(tok, V, ctx=ctx)
                 @ T.SISOVariable(id="z") @ T.GaussianLikelihood(y=y, var=0.1, ctx=ctx)).to_model()
        ep = T.ExpectationPropagation(model, ctx=ctx).iterate(max_iter=200, callback=T.EarlyStoppingEP(tol=1e-6, max_increase=np.inf), **kw)
        assert ep.status[0] == 1, kw
        r.append(ep.get_variables_data()["x"]["r"].reshape(-1))
        sweeps.append(int(ep.n_iter_instance[0]))
    assert sweeps[0] < sweeps[1]                                       # the bound is the slower of the two
    assert np.linalg.norm(r[0] - r[1]) < 1e-4 * np.linalg.norm(r[0])
