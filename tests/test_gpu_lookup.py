"""GPU: the lookup channel against its definitions in 64 bits.

Tolerances count roundings.  The kernels compute in double (u = 2^-53) and round once to the element type (half a step,
eps / 2).  A sum of c terms is off by at most (c - 1) u times the sum of their magnitudes on either side, a quotient, product
or sum by u each; the precision a' of a message is a ratio of sums of K positive terms of at most 8 operations, so it is off
by at most 2 (K + 8) u relative, in the kernel; the definition takes it in rational numbers and rounds once.  The bounds
below take 2 (c + 2 K + 32) u of the sum of magnitudes of every term of a formula: both sides' share."""
import ctypes as C

import numpy as np
import pytest

from oracle import tramp_oracle as orc
from tests.lookup_plain import LookupFactor, dense_of, zipf_tokens

pytestmark = pytest.mark.gpu
U = 2.0**-53

# V, positions, D, zipf exponent, padded share
SHAPES = [(1, 1, 1, 0.0, 0.0), (1, 5, 3, 0.0, 0.0), (7, 1, 1, 0.0, 0.0), (50, 200, 1, 1.0, 0.1), (33, 257, 5, 1.0, 0.2),
          (64, 1000, 64, 1.0, 0.0), (10, 5000, 16, 0.5, 0.05), (1000, 10, 4, 0.0, 0.0), (3, 20011, 2, 0.3, 0.0),
          (1, 70001, 1, 0.0, 0.5), (300, 900, 260, 1.2, 0.0), (40, 300, 1030, 1.0, 0.3), (4099, 30011, 1, 1.1, 0.0),
          (20, 4, 8, 0.0, 1.0), (513, 2048, 12, 0.8, 0.0), (2, 9000, 130, 0.0, 0.0),
          (20, 177, 107, 0.9, 0.1), (2, 90, 260, 0.0, 0.0), (3, 150, 1100, 0.1, 0.0), (9, 2000, 18, 0.0, 0.2)]


def make(T, ctx, shape, dtype, batch, scale, seed=0):
    V, n, D, z, pad = shape
    rs = np.random.RandomState(seed + V + 7 * n + 13 * D)
    tok = zipf_tokens(rs, V, n, z, pad)
    ch = T.LookupChannel(tok, V, dim=D, scale=scale, padding_index=-1, dtype=dtype, ctx=ctx)
    draw = lambda m: rs.standard_normal((batch, m)).astype(dtype)            # noqa: E731
    return ch, LookupFactor(tok, V, D, scale), rs, draw(V * D), draw(n * D)


def eps2(dtype):
    return np.finfo(dtype).eps / 2


@pytest.mark.parametrize("dtype", [np.float64, np.float32])
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "x".join(map(str, s[:3])))
def test_lookup_and_gradient(ctx, shape, dtype):
    import tramp_amd as T
    for batch, scale in ((1, 1.0), (3, -1.7)):
        ch, ref, rs, z, x = make(T, ctx, shape, dtype, batch, scale)
        zd, xd = ctx.array(z, dtype), ctx.array(x, dtype)
        X, G = ch.lookup(zd).get(), ch.gradient(xd).get()
        cmax = ref.count.max()
        for b in range(batch):
            want = ref.lookup(z[b]).reshape(-1)
            assert np.array_equal(X[b] == 0, want == 0)
            assert (np.abs(X[b] - want) <= (eps2(dtype) + 2 * U) * np.abs(want)).all()
            want = ref.gradient(x[b]).reshape(-1)
            mag = np.abs(scale) * LookupFactor(ref.tok, ref.V, ref.D, 1.0).gradient(np.abs(x[b])).reshape(-1)
            assert (np.abs(G[b] - want) <= eps2(dtype) * np.abs(want) + 2 * (cmax + 2) * U * mag).all()
        # the adjoint identity <lookup z, x> = <z, gradient x> and, the map being linear, its difference quotient
        left, right = np.sum(X.astype(float) * x), np.sum(z.astype(float) * G)
        size = np.sum(np.abs(X.astype(float) * x)) + np.sum(np.abs(z.astype(float) * G))
        assert abs(left - right) <= (2 * eps2(dtype) + (cmax + x.size + z.size + 8) * U) * size + 1e-300
        dz = rs.standard_normal(z.shape).astype(dtype)
        z2 = (z.astype(float) + dz).astype(dtype)
        diff = ch.lookup(ctx.array(z2, dtype)).get().astype(float) - X
        want = np.stack([ref.lookup(z2[b].astype(float) - z[b]).reshape(-1) for b in range(batch)])
        lim = (eps2(dtype) + 4 * U) * abs(scale) * np.stack([LookupFactor(ref.tok, ref.V, ref.D, 1.0).lookup(np.abs(z2[b]).astype(float) + np.abs(z[b])).reshape(-1)
                                                         for b in range(batch)])
        assert (np.abs(diff - want) <= lim).all()


def magnitudes(ref, az, bz, ax, bx, a, direction):
    "sum of the magnitudes of the terms of b'"
    lik, prec = (ax * ref.s**2 * ref.count)[:, None], ref._prec(az, ax)[:, None]
    g = abs(ref.s) * LookupFactor(ref.tok, ref.V, ref.D, 1.0).gradient(np.abs(bx.astype(float)))
    zz = np.abs(bz.astype(float)).reshape(ref.V, ref.D)
    if direction == "backward":
        return ((g * (az + a) + zz * (a + lik)) / prec).reshape(-1)
    r = np.zeros((ref.T, ref.D))
    r[ref.at] = abs(ref.s) * ((zz + g) / prec)[ref.tok[ref.at]]
    return r.reshape(-1) * (ax + a) + np.abs(bx.astype(float))


@pytest.mark.parametrize("dtype", [np.float64, np.float32])
@pytest.mark.parametrize("direction", ["forward", "backward"])
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "x".join(map(str, s[:3])))
def test_messages(ctx, shape, direction, dtype):
    import tramp_amd as T
    batch, scale = 4, 1.3
    ch, ref, rs, z, x = make(T, ctx, shape, dtype, batch, scale)
    az, ax = np.array([0.7, 1e-3, 2.0, 40.0]), np.array([1.9, 3e2, 0.0, 1e-4])
    n = x.shape[1] if direction == "forward" else z.shape[1]
    message = getattr(ch, f"compute_{direction}_message")
    posterior = getattr(ch, f"compute_{direction}_posterior")
    a_d, b_d = message(ctx.scalars(az), ctx.array(z, dtype), ctx.scalars(ax), ctx.array(x, dtype))
    r_d, v_d = posterior(ctx.scalars(az), ctx.array(z, dtype), ctx.scalars(ax), ctx.array(x, dtype))
    a0, b0 = rs.uniform(0.1, 2.0, batch), rs.standard_normal((batch, n)).astype(dtype)
    old_a, old_b = ctx.scalars(a0), ctx.array(b0, dtype)
    message(ctx.scalars(az), ctx.array(z, dtype), ctx.scalars(ax), ctx.array(x, dtype), out_a=old_a, out_b=old_b, damping=0.3,
            old_a=old_a, old_b=old_b)                                        # in place
    A, B, R, Vv, DA, DB = a_d.get(), b_d.get(), r_d.get(), v_d.get(), old_a.get(), old_b.get()
    K = np.unique(ref.count).size
    for i in range(batch):
        ra, rb = getattr(ref, direction)(az[i], z[i], ax[i], x[i])
        rel_a = 2 * (K + 8) * U
        assert abs(A[i] - ra) <= 2 * rel_a * ra + 1e-300, (i, A[i], ra)
        k = 2 * (ref.count.max() + 2 * K + 32) * U
        mag = magnitudes(ref, az[i], z[i], ax[i], x[i], ra, direction)
        assert (np.abs(B[i] - rb) <= eps2(dtype) * np.abs(rb) + k * mag).all(), i
        assert abs(DA[i] - (0.3 * a0[i] + 0.7 * ra)) <= 2 * rel_a * (a0[i] + ra)
        want = 0.3 * b0[i].astype(float) + 0.7 * rb
        assert (np.abs(DB[i] - want) <= eps2(dtype) * np.abs(want) + k * (mag + np.abs(b0[i]))).all()
        # r = (z + g) / prec: c additions, a product with s, a sum, a quotient (as a product with 1 / prec) and the product with s,
        # each off by u of its magnitude, which (|z| + |g|) / prec bounds.  (Not |b'|'s magnitude over a + a': that of a row nobody
        # reads is |z| a' / az, far below |r| (az + a').)
        mean = ref.mean(az[i], z[i], ax[i], x[i])
        size = (np.abs(z[i].astype(float)).reshape(ref.V, ref.D) + abs(ref.s) * LookupFactor(ref.tok, ref.V, ref.D, 1.0).gradient(
            np.abs(x[i].astype(float)))) / ref._prec(az[i], ax[i])[:, None]
        if direction == "forward":
            at = np.maximum(ref.tok, 0)
            mean, size = (np.where(ref.tok[:, None] >= 0, abs(ref.s) * q[at], 0.0) for q in (mean * np.sign(ref.s), size))
        lim = 2 * (ref.count.max() + 8) * U * size.reshape(-1)
        assert (np.abs(R[i] - mean.reshape(-1)) <= eps2(dtype) * np.abs(mean.reshape(-1)) + lim).all()
        v = float(getattr(ref, direction + "_variance")(az[i], ax[i]))
        assert abs(Vv[i] - v) <= rel_a * v
        assert getattr(ch, f"compute_{direction}_variance")(az[i], ax[i]) == pytest.approx(v, rel=rel_a)
        assert ch.compute_n_eff(az[i], ax[i]) == pytest.approx(ref.n_eff(az[i], ax[i]), rel=2 * rel_a, abs=0)


@pytest.mark.parametrize("dtype", [np.float64, np.float32])
def test_log_partition_and_its_gradient(ctx, dtype):
    "A of LinearChannel; dA/dbz is the posterior mean: a central difference of a quadratic is exact up to rounding"
    import tramp_amd as T
    for shape in SHAPES:
        ch, ref, rs, z, x = make(T, ctx, shape, dtype, 2, 0.8)
        az, ax = np.array([0.7, 3.0]), np.array([1.9, 0.0])
        A = ch.compute_log_partition(ctx.scalars(az), ctx.array(z, dtype), ctx.scalars(ax), ctx.array(x, dtype)).ravel()
        for i in range(2):
            want = ref.log_partition(az[i], z[i], ax[i], x[i])
            h = np.abs(z[i].astype(float)).reshape(ref.V, ref.D) + 0.8 * LookupFactor(ref.tok, ref.V, ref.D, 1.0).gradient(np.abs(x[i]).astype(float))
            prec = ref._prec(az[i], ax[i])
            mag = 0.5 * np.sum(h**2 / prec[:, None]) + 0.5 * ref.D * np.sum(np.abs(np.log(2 * np.pi / prec)) + 2)
            assert abs(A[i] - want) <= 2 * (z.shape[1] + 2 * ref.count.max() + 16) * U * mag
        step = np.zeros_like(z)
        at = rs.randint(z.shape[1])
        step[:, at] = 0.25
        up = ch.compute_log_partition(ctx.scalars(az), ctx.array(z + step, dtype), ctx.scalars(ax), ctx.array(x, dtype)).ravel()
        dn = ch.compute_log_partition(ctx.scalars(az), ctx.array(z - step, dtype), ctx.scalars(ax), ctx.array(x, dtype)).ravel()
        span = (z + step).astype(float)[:, at] - (z - step)[:, at]            # as the element type holds them
        for i in range(2):
            r = ref.mean(az[i], z[i], ax[i], x[i]).reshape(-1)[at]
            # (A(b + s) - A(b - s')) / (s + s') = r + (s - s') / (2 prec): s = s' up to the element type's rounding
            slack = 4 * (z.shape[1] + 2 * ref.count.max() + 16) * U * (mag + 1) / 0.5 + 4 * eps2(dtype) * (abs(z[i, at]) + 0.25) / ref._prec(az[i], ax[i]).min()
            assert abs((up[i] - dn[i]) / span[i] - r) <= slack


def test_host_arrays_shapes_and_extremes(ctx):
    import tramp_amd as T
    rs = np.random.RandomState(5)
    tok = np.array([[3, 0, 9], [1, 9, 3]], dtype=np.int64)
    ch = T.LookupChannel(tok, 4, dim=2, scale=2.0, padding_index=9, ctx=ctx)
    z = rs.standard_normal((4, 2))
    x = ch.sample(z)
    assert x.shape == (2, 3, 2) and np.array_equal(x, np.where((tok == 9)[..., None], 0.0, 2.0 * z[np.minimum(tok, 3)]))
    assert ch.lookup(np.stack([z, -z])).shape == (2, 2, 3, 2)
    g = ch.gradient(x)
    assert g.shape == (4, 2) and np.array_equal(g[2], [0, 0])
    a, b = ch.compute_forward_message(1.0, z, 2.0, x)
    assert isinstance(a, float) and b.shape == x.shape
    a, b = ch.compute_backward_message(1.0, z, 2.0, x)
    assert isinstance(a, float) and b.shape == z.shape
    assert isinstance(ch.compute_log_partition(1.0, z, 2.0, x), float)
    assert ch.second_moment(0.5) == 0.5 * 4.0 * 4 / 6
    for bad in (z[:3], z.T, x, np.zeros(3)):
        with pytest.raises(ValueError):
            ch.lookup(bad)
    with pytest.raises(ValueError):
        ch.compute_forward_message(1.0, z, 2.0, np.stack([x, x]))
    flat = T.LookupChannel(tok.ravel(), 4, padding_index=9, ctx=ctx)
    assert flat.sample(z[:, 0]).shape == (6,)
    # all positions padded: W = 0; the table's message is flat, the positions' one pins x to zero
    none = T.LookupChannel(np.full(5, -1), 3, padding_index=-1, ctx=ctx)
    a, b = none.compute_backward_message(1.5, np.ones(3), 2.0, np.ones(5))
    assert a == 1e-11 and np.abs(b).max() < 1e-10
    a, b = none.compute_forward_message(1.5, np.ones(3), 2.0, np.ones(5))
    assert a == 1e11 and np.array_equal(b, -np.ones(5))
    # az = 0: rows without positions stay finite in the message to the table (az is floored at 1e-11)
    one = T.LookupChannel([1, 1], 3, ctx=ctx)
    a, b = one.compute_backward_message(0.0, np.zeros(3), 2.0, np.ones(2))
    assert np.isfinite(a) and np.isfinite(b).all()
    # infinities and NaN: they reach the rows that read them and no others
    xs = np.array([np.inf, 1.0, np.nan, 2.0])
    G = T.LookupChannel([0, 1, 2, 1], 4, ctx=ctx).gradient(xs)
    assert G[0] == np.inf and G[1] == 3.0 and np.isnan(G[2]) and G[3] == 0.0
    zs = np.array([np.nan, 1.0, np.inf])
    X = T.LookupChannel([1, 7, 2], 3, padding_index=7, ctx=ctx).lookup(zs)
    assert X[0] == 1.0 and X[1] == 0.0 and X[2] == np.inf
    # a NaN at a padded position touches no row
    G = T.LookupChannel([0, 7], 2, padding_index=7, ctx=ctx).gradient(np.array([1.0, np.nan]))
    assert np.array_equal(G, [1.0, 0.0])


@pytest.mark.parametrize("dtype", [np.float64, np.float32])
def test_views_that_are_not_aligned(ctx, dtype):
    "rows of larger arrays with odd lengths: every 4- or 8-byte boundary gives the same bits"
    import tramp_amd as T
    rs = np.random.RandomState(3)
    tok = zipf_tokens(rs, 37, 501, 1.0, 0.1)
    for D in (1, 3, 8, 64):
        ch = T.LookupChannel(tok, 37, dim=D, scale=1.5, padding_index=-1, dtype=dtype, ctx=ctx)
        z, x = rs.standard_normal(37 * D).astype(dtype), rs.standard_normal(501 * D).astype(dtype)
        want = None
        for shift in (0, 1, 2, 3):
            big = lambda v: T.DeviceArray(ctx, v.shape, dtype, ptr=keep[-1].ptr + shift * v.itemsize, owner=False)   # noqa: E731
            keep, views = [], []
            for v in (z, x, z, x, z):
                keep.append(ctx.array(np.concatenate([np.zeros(shift, dtype), v, np.zeros(4, dtype)]), dtype))
                views.append(big(v))
            zz, xx, gout, xout, bout = views
            ch.lookup(zz, out=xout)
            ch.gradient(xx, out=gout)
            ch.compute_backward_message(ctx.scalars(0.7), zz, ctx.scalars(1.1), xx, out_b=bout)
            a, f = ch.compute_forward_message(ctx.scalars(0.7), zz, ctx.scalars(1.1), xx)
            got = [xout.get(), gout.get(), bout.get(), f.get()]
            ends = [k.get()[shift + len(v):] for k, v in zip(keep, (z, x, z, x, z))]
            assert all(np.array_equal(e, np.zeros(4, dtype)) for e in ends)   # nothing written behind
            if want is None:
                want = got
            for u, w in zip(got, want):
                assert np.array_equal(u, w)


def test_many_instances_and_no_instance_mixing(ctx):
    import tramp_amd as T
    rs = np.random.RandomState(8)
    tok = zipf_tokens(rs, 19, 70, 1.0, 0.1)
    ch = T.LookupChannel(tok, 19, dim=3, padding_index=-1, ctx=ctx)
    B = 301
    z, x = rs.standard_normal((B, 57)), rs.standard_normal((B, 210))
    az, ax = rs.uniform(0.5, 2, B), rs.uniform(0.1, 3, B)
    a, b = ch.compute_forward_message(ctx.scalars(az), ctx.array(z), ctx.scalars(ax), ctx.array(x))
    A, Bn = a.get(), b.get()
    for i in (0, 7, 300):
        a1, b1 = ch.compute_forward_message(ctx.scalars(az[i]), ctx.array(z[i]), ctx.scalars(ax[i]), ctx.array(x[i]))
        assert a1.get()[0] == A[i] and np.array_equal(b1.get(), Bn[i])


def test_captured_calls_replay_and_share_workspaces(ctx):
    "two graphs and eager calls between the replays, all on one context: every replay gives the eager bits"
    import tramp_amd as T
    rs = np.random.RandomState(11)
    sets = []
    for V, n, D, dt in ((50, 20000, 3, np.float64), (400, 3000, 64, np.float32)):
        tok = zipf_tokens(rs, V, n, 1.0, 0.1)
        ch = T.LookupChannel(tok, V, dim=D, padding_index=-1, dtype=dt, ctx=ctx)
        s = dict(ch=ch, z=ctx.array(rs.standard_normal((2, V * D)), dt), x=ctx.array(rs.standard_normal((2, n * D)), dt),
                 az=ctx.scalars([0.5, 1.0]), ax=ctx.scalars([2.0, 0.3]), oa=ctx.empty((2,)), ob=ctx.empty((2, n * D), dt),
                 pa=ctx.empty((2,)), pb=ctx.empty((2, V * D), dt))

        def calls(s):
            s["ch"].compute_forward_message(s["az"], s["z"], s["ax"], s["x"], out_a=s["oa"], out_b=s["ob"])
            s["ch"].compute_backward_message(s["az"], s["z"], s["ax"], s["x"], out_a=s["pa"], out_b=s["pb"])
        calls(s)
        s["want"] = [s[k].get() for k in ("oa", "ob", "pa", "pb")]
        sets.append(s)
    for s in sets:
        ctx._call("tramp_graph_begin")
        calls(s)
        s["graph"] = C.c_void_p()
        ctx._call("tramp_graph_end", C.byref(s["graph"]))
    try:
        for rep in range(4):
            for s in sets:
                for k in ("oa", "ob", "pa", "pb"):
                    s[k].fill(-1.0)
                ctx._call("tramp_graph_launch", s["graph"])
                got = [s[k].get() for k in ("oa", "ob", "pa", "pb")]
                assert all(np.array_equal(g, w) for g, w in zip(got, s["want"]))
                s["ch"].gradient(s["x"])
            ctx.sync()
    finally:
        for s in sets:
            ctx._call("tramp_graph_destroy", s["graph"])


@pytest.mark.parametrize("V, n, D, B, zipf, pad, dtype", [(700001, 600000, 1, 1, None, 0.0, np.float64), (3000, 90000, 7, 1, 1.1, 0.1, np.float64),
                                                          (500, 80000, 1, 16, 1.0, 0.2, np.float32), (2500, 40001, 3, 16, 1.2, 0.1, np.float32),
                                                          (20000, 30000, 5, 8, 0.5, 0.0, np.float64), (300, 200000, 33, 3, 1.0, 0.1, np.float32),
                                                          (9001, 3001, 40, 3, 0.3, 0.1, np.float64), (6000, 2501, 96, 8, 0.0, 0.0, np.float32),
                                                          (500, 20000, 66, 8, 0.0, 0.05, np.float32), (300, 12000, 140, 5, 0.0, 0.0, np.float64)])
def test_larger_messages(ctx, V, n, D, B, zipf, pad, dtype):
    "the forms that only larger calls take: by position, heavy runs, instances by XCD, no token twice; same tolerances"
    import tramp_amd as T
    rs = np.random.RandomState(1)
    tok = rs.permutation(V)[:n] if zipf is None else zipf_tokens(rs, V, n, zipf, pad)
    ch = T.LookupChannel(tok, V, dim=D, scale=0.7, padding_index=-1, dtype=dtype, ctx=ctx)
    ref = LookupFactor(tok, V, D, 0.7)
    z, x = rs.standard_normal((B, V * D)).astype(dtype), rs.standard_normal((B, n * D)).astype(dtype)
    az, ax = rs.uniform(0.5, 2, B), rs.uniform(0.1, 3, B)
    args = ctx.scalars(az), ctx.array(z, dtype), ctx.scalars(ax), ctx.array(x, dtype)
    K = np.unique(ref.count).size
    k = 2 * (ref.count.max() + 2 * K + 32) * U
    for direction in ("forward", "backward"):
        a, b = getattr(ch, f"compute_{direction}_message")(*args)
        a2, b2 = getattr(ch, f"compute_{direction}_message")(*args)
        assert np.array_equal(a.get(), a2.get()) and np.array_equal(b.get(), b2.get())       # the same bits every time
        damped_a, damped_b = ctx.scalars(np.ones(B)), ctx.zeros(b.shape, dtype)
        getattr(ch, f"compute_{direction}_message")(*args, out_a=damped_a, out_b=damped_b, damping=0.5, old_a=damped_a, old_b=damped_b)
        r, _ = getattr(ch, f"compute_{direction}_posterior")(*args)
        A, Bn, R, Db = a.get(), b.get(), r.get(), damped_b.get()
        for i in {0, B - 1}:
            ra, rb = getattr(ref, direction)(az[i], z[i], ax[i], x[i])
            mag = magnitudes(ref, az[i], z[i], ax[i], x[i], ra, direction)
            assert abs(A[i] - ra) <= 4 * (K + 8) * U * ra
            assert (np.abs(Bn[i] - rb) <= eps2(dtype) * np.abs(rb) + k * mag).all()
            assert (np.abs(Db[i] - 0.5 * rb) <= eps2(dtype) * np.abs(0.5 * rb) + k * mag).all()
            own = z[i] if direction == "backward" else x[i]
            a_in = az[i] if direction == "backward" else ax[i]
            # b' = r (a + a') - b on the posterior the same call gives, which is rounded once more
            lim = k * mag + eps2(dtype) * (np.abs(rb) + np.abs(R[i].astype(float)) * (a_in + ra)) + 4 * U * (np.abs(R[i].astype(float)) * (a_in + ra) + np.abs(own))
            assert (np.abs(Bn[i] - (R[i].astype(float) * (a_in + ra) - own)) <= lim).all()


@pytest.mark.parametrize("dtype", [np.float64, np.float32])
@pytest.mark.parametrize("V, n, D, pad", [(5003, 1201, 33, 0.1), (1203, 2001, 64, 0.0), (70, 9, 1030, 0.3), (9, 9, 16, 0.0), (4001, 3, 17, 0.0), (3001, 40, 1, 0.0),
                                          (6, 5, 130, 1.0)])
def test_rows_that_few_positions_read(ctx, V, n, D, pad, dtype):
    "tables of rows read once or never: every component is written, and the sums of one position are that position's"
    import tramp_amd as T
    rs = np.random.RandomState(V + n)
    tok = zipf_tokens(rs, V, n, 0.2, pad)
    ch, ref = T.LookupChannel(tok, V, dim=D, scale=-0.6, padding_index=-1, dtype=dtype, ctx=ctx), LookupFactor(tok, V, D, -0.6)
    B = 2
    z, x = rs.standard_normal((B, V * D)).astype(dtype), rs.standard_normal((B, n * D)).astype(dtype)
    unset = lambda m: ctx.array(np.full((B, m), np.nan), dtype)            # noqa: E731
    G = ch.gradient(ctx.array(x, dtype), out=unset(V * D)).get()
    plain = LookupFactor(tok, V, D, 1.0)
    az, ax = np.array([0.8, 5.0]), np.array([2.0, 0.1])
    args = ctx.scalars(az), ctx.array(z, dtype), ctx.scalars(ax), ctx.array(x, dtype)
    k = 2 * (ref.count.max() + 2 * np.unique(ref.count).size + 32) * U
    for b in range(B):
        want = ref.gradient(x[b]).reshape(-1)
        mag = 0.6 * plain.gradient(np.abs(x[b])).reshape(-1)
        assert (np.abs(G[b] - want) <= eps2(dtype) * np.abs(want) + 2 * (ref.count.max() + 2) * U * mag).all()
    assert (G.reshape(B, V, D)[:, ref.count == 0] == 0).all()
    for direction, m in (("forward", n * D), ("backward", V * D)):
        got = getattr(ch, f"compute_{direction}_message")(*args, out_a=ctx.scalars(np.ones(B)), out_b=unset(m))[1].get()
        b0 = rs.standard_normal((B, m)).astype(dtype)
        old = ctx.array(b0, dtype)
        damped = getattr(ch, f"compute_{direction}_message")(*args, out_a=ctx.scalars(np.ones(B)), out_b=unset(m), damping=0.4,
                                                             old_a=ctx.scalars(np.ones(B)), old_b=old)[1].get()
        assert np.array_equal(old.get(), b0)
        for b in range(B):
            ra, rb = getattr(ref, direction)(az[b], z[b], ax[b], x[b])
            mag = magnitudes(ref, az[b], z[b], ax[b], x[b], ra, direction)
            assert (np.abs(got[b] - rb) <= eps2(dtype) * np.abs(rb) + k * mag).all()
            want = 0.4 * b0[b].astype(float) + 0.6 * rb
            assert (np.abs(damped[b] - want) <= eps2(dtype) * np.abs(want) + k * (mag + np.abs(b0[b]))).all()


@pytest.mark.parametrize("dtype", [np.float64, np.float32])
@pytest.mark.parametrize("V, n, D, heavy, pad", [(1, 1, 1, 0, 0), (40, 25, 5, 0, 0), (2000, 1201, 33, 0, 0), (30, 30, 260, 0, 0), (50, 41, 6, 3, 4),
                                                 (700001, 600000, 1, 0, 0), (500000, 400000, 7, 2200, 0)])
def test_a_position_alone_in_its_run_keeps_its_digits(ctx, V, n, D, heavy, pad, dtype):
    """az far below ax scale^2: r (a + a') and b are both about b, the message is what bz has left.  Of a run of one it is
    [s (ax + a') bz + (s^2 a' - az) bx] / prec, two terms that do not cancel: the kernel's a' is off by 2 (K + 8) u relative, a product or
    quotient by u each, which 2 (K + 16) u of the terms' magnitudes holds.  The definition is taken in 64 bits of mantissa."""
    import tramp_amd as T
    rs = np.random.RandomState(V + n + D)
    s = 0.7
    tok = rs.permutation(V)[:n]
    tok[:heavy], tok[n - pad:] = V - 1, -1
    ch, ref = T.LookupChannel(tok, V, dim=D, scale=s, padding_index=-1, dtype=dtype, ctx=ctx), LookupFactor(tok, V, D, s)
    az, ax = np.array([1.0, 0.3]), np.array([1e9, 3e6])
    z = rs.standard_normal((2, V * D)).astype(dtype)
    x = (ax[:, None] * rs.standard_normal((2, n * D))).astype(dtype)
    a_d, b_d = ch.compute_forward_message(ctx.scalars(az), ctx.array(z, dtype), ctx.scalars(ax), ctx.array(x, dtype))
    got = b_d.get().reshape(2, n, D)
    K = np.unique(ref.count).size
    one = np.flatnonzero((tok >= 0) & (ref.count[np.maximum(tok, 0)] == 1))
    L = np.longdouble
    for b in range(2):
        ra = ref._a(ref.forward_variance(az[b], ax[b]), ax[b])
        zz, xx = z[b].reshape(V, D)[tok[one]].astype(L), x[b].reshape(n, D)[one].astype(L)
        prec = L(az[b]) + L(ax[b]) * L(s) * L(s)
        kz, kx = L(s) * (L(ax[b]) + L(ra)) / prec, (L(s) * L(s) * L(ra) - L(az[b])) / prec
        want = kz * zz + kx * xx
        mag = np.abs(kz * zz) + np.abs(xx) * (L(s) * L(s) * L(ra) + L(az[b])) / prec
        assert (np.abs(got[b, one] - want) <= eps2(dtype) * np.abs(want) + 2 * (K + 16) * U * mag).all(), b


def test_a_precision_that_is_nan_stays_one(ctx):
    import tramp_amd as T
    ch = T.LookupChannel([0, 1, 1], 3, ctx=ctx)
    for az, ax in ((np.nan, 1.0), (1.0, np.nan)):
        for m in (ch.compute_forward_message, ch.compute_backward_message):
            a, _ = m(ctx.scalars(az), ctx.array(np.ones(3)), ctx.scalars(ax), ctx.array(np.ones(3)))
            assert np.isnan(a.get()).all()


def test_offsets_beyond_32_bits(ctx):
    "2.2e9 components: rows at the far end of x against the definition, the sums against the counts"
    import tramp_amd as T
    n, D = 2200000, 1024
    tok = np.arange(n) % 3
    tok[-1] = -1
    ch = T.LookupChannel(tok, 3, dim=D, scale=2.0, padding_index=-1, dtype=np.float32, ctx=ctx)
    rs = np.random.RandomState(0)
    z = rs.randint(-8, 9, (3, D)).astype(np.float32)                   # small integers: every sum below is exact
    zd = ctx.array(z.reshape(1, -1), np.float32)
    x = ch.lookup(zd)
    row = lambda buf, t: T.DeviceArray(ctx, (D,), np.float32, ptr=buf.ptr + 4 * t * D, owner=False).get()      # noqa: E731
    for t in (0, 1, 2**21 - 1, 2**21, 2**21 + 1, n - 3, n - 2):
        assert np.array_equal(row(x, t), 2 * z[tok[t]])
    assert np.array_equal(row(x, n - 1), np.zeros(D, np.float32))
    count = np.bincount(tok[:-1], minlength=3)
    g = ch.gradient(x).get().reshape(3, D)
    assert np.array_equal(g, (4.0 * count[:, None] * z.astype(float)).astype(np.float32))
    a, b = ch.compute_forward_message(ctx.scalars(1.0), zd, ctx.scalars(0.5), x)
    ref = LookupFactor(tok, 3, 1, 2.0)
    ra = ref._a(ref.forward_variance(1.0, 0.5), 0.5)
    prec = 1.0 + 0.5 * 4 * count
    mean = 2 * (z + 4.0 * count[:, None] * z) / prec[:, None]
    for t in (0, 2**21, n - 2):
        want = mean[tok[t]] * (0.5 + ra) - 2 * z[tok[t]]
        assert np.abs(row(b, t) - want).max() <= 2**-23 * np.abs(want).max() + 1e-9 * np.abs(mean).max() * (0.5 + ra)
    assert np.array_equal(row(b, n - 1), np.zeros(D, np.float32)) and a.get()[0] == pytest.approx(ra, rel=1e-12)


def test_more_instances_than_one_axis_of_a_grid_holds(ctx):
    "65528 instances of 65700 rows: 1.68e7 workgroups of 256; every component of the 17 GB is written, one per instance not zero"
    import tramp_amd as T
    B, V = 65528, 65700
    ch = T.LookupChannel([V - 3], V, scale=2.0, dtype=np.float32, ctx=ctx)
    x = np.arange(1, B + 1, dtype=np.float32)[:, None]
    g = ctx.full((B, V), np.nan, np.float32)
    ch.gradient(ctx.array(x, np.float32), out=g)
    assert np.array_equal(T.ArrayGroup([g]).norm().get(), 2.0 * x[:, 0])
    for b in (0, 1, B // 2, B - 1):
        row = T.DeviceArray(ctx, (V,), np.float32, ptr=g.ptr + 4 * b * V, owner=False).get()
        assert row[V - 3] == 2.0 * x[b, 0] and np.count_nonzero(row) == 1
    X = ch.lookup(g).get()
    assert np.array_equal(X, 4.0 * x)


def test_refusals_on_the_device(ctx):
    import tramp_amd as T
    ch = T.LookupChannel([0, 1, 1], 2, ctx=ctx)
    z, x = ctx.array(np.ones(2)), ctx.array(np.ones(3))
    with pytest.raises(T._lib.TrampHipError):
        ctx._call("tramp_lookup_apply", ch._handle, 1, z.ptr, z.ptr)
    with pytest.raises(T._lib.TrampHipError):
        ctx._call("tramp_lookup_gradient", ch._handle, 1, x.ptr, x.ptr)
    with pytest.raises(T._lib.TrampHipError):
        ctx._call("tramp_lookup_apply", ch._handle, 65536, z.ptr, x.ptr)
    with pytest.raises(ValueError):
        ch.lookup(z, out=ctx.empty((1, 4)))
    with pytest.raises(ValueError):
        ch.lookup(z, out=np.empty(3))
    with pytest.raises(TypeError):
        ch.lookup(ctx.array(np.ones(2), np.float32))
    with pytest.raises(ValueError):
        ch.gradient(z)
    a = ctx.scalars(1.0)
    with pytest.raises(T._lib.TrampHipError):
        ch.compute_backward_message(a, z, a, x, out_b=z)
    for kw in (dict(out_a=ctx.empty((2,))), dict(out_b=ctx.empty((3,))), dict(damping=0.5), dict(damping=0.5, old_a=a, old_b=x),
               dict(damping=0.5, old_a=ctx.empty((2,)), old_b=ctx.empty((2,))), dict(out_a=ctx.empty((1,), np.float32))):
        with pytest.raises(ValueError):
            ch.compute_backward_message(a, z, a, x, **kw)
    big = ctx.zeros((12,))
    part = lambda lo, n: T.DeviceArray(ctx, (n,), np.float64, ptr=big.ptr + 8 * lo, owner=False)       # noqa: E731
    for call in (lambda: ch.lookup(part(0, 2), out=part(1, 3)), lambda: ch.gradient(part(2, 3), out=part(1, 2)),
                 lambda: ch.compute_forward_message(a, part(0, 2), a, part(2, 3), out_b=part(4, 3)),
                 lambda: ch.compute_forward_message(a, part(0, 2), a, part(2, 3), out_b=part(6, 3), damping=0.5, old_a=a, old_b=part(7, 3))):
        with pytest.raises(T._lib.TrampHipError):
            call()
    assert np.array_equal(big.get(), np.zeros(12))
    with pytest.raises(T._lib.TrampHipError):
        ctx._call("tramp_lookup_message", ch._handle, 0, 1, a.ptr, z.ptr, a.ptr, x.ptr, 0.5, None, None, a.ptr, ctx.empty(3).ptr, None, None)
    old = ctx.zeros((1, 3))                                            # the posterior over the old message
    with pytest.raises(T._lib.TrampHipError):
        ctx._call("tramp_lookup_message", ch._handle, T._lib.FWD, 1, a.ptr, z.ptr, a.ptr, x.ptr, 0.5, a.ptr, old.ptr, a.ptr,
                  ctx.empty((1, 3)).ptr, old.ptr, None)
    h = C.c_void_p()
    bad = np.array([0, 5], dtype=np.int32)
    for args in ((1, 2, 1, 2, bad.ctypes.data, 1.0), (1, 2, 0, 2, bad.ctypes.data, 1.0), (7, 9, 1, 2, bad.ctypes.data, 1.0),
                 (1, 9, 1, 2, bad.ctypes.data, float("nan")), (1, 9, 1, 2, None, 1.0)):
        with pytest.raises(T._lib.TrampHipError):
            ctx._call("tramp_lookup_create", *args, C.byref(h))
    other = T.Context(0)
    try:
        with pytest.raises(ValueError):
            ch.lookup(other.array(np.ones(2)))
    finally:
        other.close()


@pytest.mark.parametrize("V, n, D, B", [(20, 30, 3, 4), (9, 5, 1, 2), (3, 9000, 2, 3), (400, 70000, 4, 3)])
def test_scalar_results_in_place_and_shifted(ctx, V, n, D, B):
    "a' or v over the precisions it is made of: the bits of the call with buffers of its own, in every form; shifted: refused"
    import tramp_amd as T
    rs = np.random.RandomState(n)
    ch = T.LookupChannel(zipf_tokens(rs, V, n, 0.6, 0.1), V, dim=D, padding_index=-1, ctx=ctx)
    z, x = ctx.array(rs.standard_normal((B, V * D))), ctx.array(rs.standard_normal((B, n * D)))
    scal = {"az": rs.uniform(0.5, 2, B), "ax": rs.uniform(0.1, 3, B), "a_old": rs.uniform(0.5, 2, B)}
    for direction, m in ((T._lib.FWD, n * D), (T._lib.BWD, V * D)):
        old = ctx.array(rs.standard_normal((B, m)))

        def run(a_new=None, v=None, shift=0):
            d = {k: ctx.array(np.concatenate([s, np.zeros(1)])) for k, s in scal.items()}
            put = lambda name: d[name].ptr + 8 * shift if name else d.setdefault("own" + str(len(d)), ctx.empty((B,))).ptr      # noqa: E731
            pa, pv, b, r = put(a_new), put(v), ctx.empty((B, m)), ctx.empty((B, m))
            ctx._call("tramp_lookup_message", ch._handle, direction, B, d["az"].ptr, z.ptr, d["ax"].ptr, x.ptr, 0.25, d["a_old"].ptr, old.ptr,
                      pa, b.ptr, r.ptr, pv)
            return [T.DeviceArray(ctx, (B,), np.float64, ptr=q, owner=False).get() for q in (pa, pv)] + [b.get(), r.get()]
        want = run()
        for over in (dict(a_new="az"), dict(a_new="ax"), dict(v="az"), dict(v="ax"), dict(v="a_old"), dict(a_new="ax", v="az")):
            for got, w in zip(run(**over), want):
                assert np.array_equal(got, w), over
            with pytest.raises(T._lib.TrampHipError):
                run(**over, shift=1)
    both = ctx.array(np.arange(1.0, 2 * B + 1))
    at = lambda i: both.ptr + 8 * i                                    # noqa: E731
    for args in ((at(0), at(B), at(1), None, None), (at(0), at(B), None, at(B - 1), None), (at(0), at(0), at(B), at(B), None),
                 (at(0), at(0), None, at(B), at(B - 1))):
        with pytest.raises(T._lib.TrampHipError):
            ctx._call("tramp_lookup_variance", ch._handle, T._lib.FWD, B, *args)
    assert np.array_equal(both.get(), np.arange(1.0, 2 * B + 1))
    out = ctx.empty((B, n * D))
    with pytest.raises(T._lib.TrampHipError):                         # a vector over the precisions
        ctx._call("tramp_lookup_message", ch._handle, T._lib.FWD, B, out.ptr + 8, z.ptr, at(0), x.ptr, 0.0, None, None, at(B), out.ptr, None, None)


# ---------------------------------------------------------------- in models
def regression(T, ctx, channel, V, y, prior="gb"):
    pri = T.GaussBernoulliPrior(size=V, rho=0.5, ctx=ctx)
    return (pri @ T.SISOVariable(id="x") @ channel @ T.SISOVariable(id="z") @ T.GaussianLikelihood(y=y, var=0.1, ctx=ctx)).to_model()


@pytest.mark.parametrize("damping, graph", [(None, False), (0.3, False), (0.3, True)])
def test_ep_matches_the_dense_channel_and_the_oracle(ctx, damping, graph):
    import tramp_amd as T
    rs = np.random.RandomState(2)
    V, n, B = 60, 150, 3
    tok = zipf_tokens(rs, V, n, 0.8, 0.1)
    W = dense_of(tok, V, 1, 1.4)
    X = np.stack([orc.gb_sample(rs, V, 0.5) for _ in range(B)])
    Y = X @ W.T + np.sqrt(0.1) * rs.standard_normal((B, n))
    lk = T.LookupChannel(tok, V, scale=1.4, padding_index=-1, ctx=ctx)
    ep = T.ExpectationPropagation(regression(T, ctx, lk, V, Y), ctx=ctx)
    ep.iterate(max_iter=20, callback=T.PassCallback(), damping=damping, graph=graph)
    r = ep.get_variables_data()["x"]["r"]
    ref = LookupFactor(tok, V, 1, 1.4)
    for b in range(B):
        res = orc.ep_chain([orc.GBPriorFactor(V, rho=0.5), ref, orc.GaussLikFactor(Y[b], 0.1)], [V, n], max_iter=20,
                           damping=damping, tol=0.0, max_increase=np.inf)
        assert np.abs(r[b] - res["r"][0]).max() < 1e-9 * np.abs(res["r"][0]).max()
    dense = T.ExpectationPropagation(regression(T, ctx, T.LinearChannel(W, ctx=ctx, svd="host"), V, Y), ctx=ctx)
    dense.iterate(max_iter=20, callback=T.PassCallback(), damping=damping)
    rd = dense.get_variables_data()["x"]["r"]
    assert np.abs(r - rd).max() < 1e-8 * np.abs(rd).max()
    np.testing.assert_allclose(ep.log_evidence(), dense.log_evidence(), rtol=1e-8)


def test_adaptive_damping_matches_the_dense_channel(ctx):
    "the step-halving search evaluates messages and log-partitions of candidates: the same trajectory as the one-hot matrix"
    import tramp_amd as T
    rs = np.random.RandomState(8)
    V, n = 40, 90
    tok = zipf_tokens(rs, V, n, 0.7, 0.1)
    W = dense_of(tok, V, 1, 1.2)
    y = W @ orc.gb_sample(rs, V, 0.5) + np.sqrt(0.1) * rs.standard_normal(n)
    r, logz = [], []
    for ch in (T.LookupChannel(tok, V, scale=1.2, padding_index=-1, ctx=ctx), T.LinearChannel(W, ctx=ctx, svd="host")):
        ep = T.ExpectationPropagation(regression(T, ctx, ch, V, y), ctx=ctx)
        ep.iterate(max_iter=6, callback=T.PassCallback(), damping="adaptive")
        r.append(ep.get_variables_data()["x"]["r"].reshape(-1))
        logz.append(ep.log_evidence())
    assert np.abs(r[0] - r[1]).max() < 1e-7 * np.abs(r[1]).max()
    assert logz[0] == pytest.approx(logz[1], rel=1e-7)


def test_one_table_read_twice_in_a_tree(ctx):
    "x feeds two lookups with tokens of their own: the exact posterior of the Gaussian model"
    import tramp_amd as T
    rs = np.random.RandomState(10)
    V, n1, n2 = 20, 70, 33
    t1, t2 = rs.randint(0, V, n1), zipf_tokens(rs, V, n2, 1.0, 0.2)
    y1, y2 = rs.standard_normal(n1), rs.standard_normal(n2)
    W1, W2 = dense_of(t1, V, 1, 1.0), dense_of(t2, V, 1, 0.5)
    want = np.linalg.solve(np.eye(V) + W1.T @ W1 / 0.2 + W2.T @ W2 / 0.4, W1.T @ y1 / 0.2 + W2.T @ y2 / 0.4)
    model = (T.GaussianPrior(size=V, ctx=ctx) @ T.SIMOVariable(id="x", n_next=2) @ (
        (T.LookupChannel(t1, V, ctx=ctx) @ T.SISOVariable(id="z1") @ T.GaussianLikelihood(y=y1, var=0.2, ctx=ctx))
        + (T.LookupChannel(t2, V, scale=0.5, padding_index=-1, ctx=ctx) @ T.SISOVariable(id="z2") @ T.GaussianLikelihood(y=y2, var=0.4, ctx=ctx)))).to_model()
    ep = T.ExpectationPropagation(model, ctx=ctx)
    ep.iterate(max_iter=500, damping=0.3, callback=T.EarlyStoppingEP(tol=1e-10, max_increase=np.inf))
    assert np.abs(ep.get_variables_data()["x"]["r"].reshape(-1) - want).max() < 1e-6


def test_state_evolution_sampling_and_tables(ctx):
    "a table of D columns, positions of two axes; SE against the dense channel of the same matrix"
    import tramp_amd as T
    rs = np.random.RandomState(4)
    V, D = 30, 3
    tok = zipf_tokens(rs, V, 40, 0.5).reshape(8, 5)
    W = dense_of(tok, V, D, 0.9)
    lk = T.LookupChannel(tok, V, dim=D, scale=0.9, ctx=ctx)
    model = (T.GaussianPrior(size=(V, D), ctx=ctx) @ T.SISOVariable(id="x") @ lk @ T.SISOVariable(id="z")
             @ T.GaussianChannel(var=0.2) @ T.SILeafVariable(id="y")).to_model()
    s = model.sample(seed=3)
    assert s["z"].shape == (8, 5, D) and np.allclose(s["z"].reshape(-1), W @ s["x"].reshape(-1), rtol=1e-15, atol=0)
    assert model.init_shapes()["z"] == (8, 5, D)
    model.init_second_moments()
    lin = orc.LinearOracle(W)
    assert model.get_second_moments()["z"] == pytest.approx(lin.second_moment(1.0), rel=1e-12)
    for az, ax in ((0.3, 2.0), (5.0, 0.0), (1.0, 40.0)):
        assert lk.compute_forward_error(az, ax, 1.0) == pytest.approx(lin.forward_variance(az, ax), rel=1e-9)
        assert lk.compute_backward_error(az, ax, 1.0) == pytest.approx(lin.backward_variance(az, ax), rel=1e-9)
    obs = model.to_observed({"y": s["y"]})
    ep = T.ExpectationPropagation(obs, ctx=ctx)
    ep.iterate(max_iter=60, damping=0.1)
    # Gaussian prior and noise: EP's fixed point is the exact posterior mean
    H = W.T @ W / 0.2 + np.eye(V * D)
    want = np.linalg.solve(H, W.T @ s["y"].reshape(-1) / 0.2)
    assert np.abs(ep.get_variables_data()["x"]["r"].reshape(-1) - want).max() < 1e-4 * np.abs(want).max()
    se = T.StateEvolution(obs)
    se.iterate(max_iter=50)
    assert 0 < se.get_variables_data()["x"]["v"] < 1


def test_a_channel_made_on_one_context_runs_on_another(ctx):
    import tramp_amd as T
    rs = np.random.RandomState(6)
    tok = zipf_tokens(rs, 20, 50, 0.5)
    y = rs.standard_normal(50)
    lk = T.LookupChannel(tok, 20, ctx=ctx)
    want = T.ExpectationPropagation(regression(T, ctx, lk, 20, y), ctx=ctx).iterate(max_iter=5, callback=T.PassCallback()).get_variables_data()["x"]["r"]
    other = T.Context(0)
    lk2 = T.LookupChannel(tok, 20, ctx=ctx)
    got = T.ExpectationPropagation(regression(T, other, lk2, 20, y), ctx=other).iterate(max_iter=5, callback=T.PassCallback()).get_variables_data()["x"]["r"]
    assert np.array_equal(want, got)
    del lk2
