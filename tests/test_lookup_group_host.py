"""Refusals of the lookup channel, of the array lists and of iterate(max_step=...) that need no device, and the plain
definitions the GPU tests compare with, checked against the dense oracle of the linear channel."""
import ctypes as C
import os
import subprocess

import numpy as np
import pytest

import tramp_amd as T
from oracle import tramp_oracle as orc
from tests.lookup_plain import LookupFactor, clip_plain, dense_of, step_plain


class HostContext:
    "stands where a context goes; the checks under test raise before any call"
    device = 0
    handle = None

    def _call(self, name, *args):
        raise AssertionError(f"{name} was reached")

    def release(self, name, handle):
        pass


def fake(ctx, shape, dtype=np.float64, ptr=4096):
    return T.DeviceArray(ctx, shape, dtype, ptr=ptr, owner=False)


@pytest.mark.parametrize("kw, error", [
    (dict(tokens=[0.5, 1.0], n_tokens=3), TypeError),
    (dict(tokens=[True, False], n_tokens=3), TypeError),
    (dict(tokens=np.zeros(0, int), n_tokens=3), ValueError),
    (dict(tokens=[0, 3], n_tokens=3), ValueError),
    (dict(tokens=[0, -1], n_tokens=3), ValueError),
    (dict(tokens=[0, -2], n_tokens=3, padding_index=-1), ValueError),
    (dict(tokens=[0, 2**40], n_tokens=3), ValueError),
    (dict(tokens=[0], n_tokens=0), ValueError),
    (dict(tokens=[0], n_tokens=3, dim=0), ValueError),
    (dict(tokens=[0], n_tokens=2**31), ValueError),
    (dict(tokens=[0], n_tokens=3, scale=0.0), ValueError),
    (dict(tokens=[0], n_tokens=3, scale=np.nan), ValueError),
    (dict(tokens=[0], n_tokens=3, scale=np.inf), ValueError),
    (dict(tokens=[0], n_tokens=3, dtype=np.float16), ValueError),
])
def test_lookup_channel_refuses(kw, error):
    with pytest.raises(error):
        T.LookupChannel(ctx=HostContext(), **kw)


def test_valid_arguments_reach_the_library():
    with pytest.raises(AssertionError, match="tramp_lookup_create"):
        T.LookupChannel([[0, 2], [7, 1]], 3, dim=2, padding_index=7, ctx=HostContext())
    with pytest.raises(AssertionError, match="tramp_lookup_create"):
        T.get_channel("lookup", tokens=np.uint8([0, 1]), n_tokens=2, ctx=HostContext())


@pytest.mark.parametrize("dtype", [np.uint8, np.uint16, np.uint32, np.uint64, np.int8, np.int16, np.int64])
def test_padded_positions_of_any_integer_type(dtype):
    "-1 where padded, also where the type cannot hold it and the table is longer than its largest value"
    seen = []

    class Recorder(HostContext):
        def _call(self, name, dt, rows, cols, n, tokens, *rest):
            seen.extend((C.c_int * n).from_address(tokens))
            raise AssertionError(name)

    last = int(np.iinfo(dtype).max)
    with pytest.raises(AssertionError, match="tramp_lookup_create"):
        T.LookupChannel(np.array([0, last, 5, 1], dtype=dtype), 70000, padding_index=last, ctx=Recorder())
    assert seen == [0, -1, 5, 1]


def test_the_largest_sizes_are_refused_before_anything_is_allocated():
    many = np.broadcast_to(np.int8(0), (2**31 - 2**16 + 1,))             # one byte of memory
    with pytest.raises(ValueError, match="exceed"):
        T.LookupChannel(many, 3, ctx=HostContext())
    for kw in (dict(n_tokens=2**31 - 2**16 + 1), dict(n_tokens=3, dim=2**31 - 2**16 + 1)):
        with pytest.raises(ValueError, match="exceed"):
            T.LookupChannel([0], ctx=HostContext(), **kw)
    with pytest.raises(AssertionError, match="tramp_lookup_create"):
        T.LookupChannel([0], 2**31 - 2**16, ctx=HostContext())


def test_array_group_refuses():
    ctx, other = HostContext(), HostContext()
    a = fake(ctx, (2, 5))
    for arrays in ([], [np.zeros((2, 5))], [a, fake(ctx, (3, 5), ptr=1 << 20)], [a, fake(ctx, (2, 5), np.float32, ptr=1 << 20)],
                   [a, fake(other, (2, 5), ptr=1 << 20)], [fake(ctx, (1, 2, 5))], [fake(ctx, (4,), np.uint8)]):
        with pytest.raises(ValueError):
            T.ArrayGroup(arrays)
    with pytest.raises(AssertionError, match="tramp_group_create"):
        T.ArrayGroup([a, fake(ctx, (2, 7), ptr=1 << 20)])


def make_group(ctx, lengths, batch=2, dtype=np.float64):
    g = T.ArrayGroup.__new__(T.ArrayGroup)
    g.ctx, g.dtype, g.batch, g.lengths, g._handle = ctx, np.dtype(dtype), batch, tuple(lengths), C.c_void_p()
    g.arrays = [fake(ctx, (batch, n)) for n in lengths]
    return g


def test_group_calls_refuse():
    ctx = HostContext()
    g = make_group(ctx, (4, 5))
    norm = fake(ctx, (2,))
    for bad in (0.0, -1.0, np.nan):
        with pytest.raises(ValueError):
            g.clip(bad, norm=norm)
        with pytest.raises(ValueError):
            g.limit_step(make_group(ctx, (4, 5)), bad, norm=norm)
    for other in (make_group(ctx, (4, 6)), make_group(ctx, (4,)), make_group(ctx, (4, 5), batch=3), make_group(ctx, (4, 5), dtype=np.float32),
                  make_group(HostContext(), (4, 5)), [1, 2]):
        with pytest.raises(ValueError):
            g.clip(1.0, out=other, norm=norm)
        with pytest.raises(ValueError):
            g.limit_step(other, 1.0, norm=norm)
    for bad_norm in (fake(ctx, (3,)), fake(ctx, (2,), np.float32), np.zeros(2), fake(HostContext(), (2,))):
        with pytest.raises(ValueError):
            g.norm(bad_norm)
    prev = make_group(ctx, (4, 5))
    with pytest.raises(ValueError):
        g.limit_step(prev, 1.0, norm=norm, a=fake(ctx, (3, 2)))
    for a in (fake(ctx, (3, 4)), fake(ctx, (3, 2), np.float32), np.zeros((3, 2))):
        with pytest.raises(ValueError):
            g.limit_step(prev, 1.0, norm=norm, a=a, a_prev=fake(ctx, (3, 2)))


def test_c_entries_refuse_a_null_context():
    lib = T._lib.load()
    h = C.c_void_p()
    assert lib.tramp_lookup_create(None, 1, 2, 1, 1, None, 1.0, C.byref(h)) == T._lib.EINVAL
    assert lib.tramp_lookup_apply(None, None, 1, None, None) == T._lib.EINVAL
    assert lib.tramp_lookup_gradient(None, None, 1, None, None) == T._lib.EINVAL
    assert lib.tramp_lookup_message(None, None, 0, 1, None, None, None, None, 0.0, None, None, None, None, None, None) == T._lib.EINVAL
    assert lib.tramp_lookup_variance(None, None, 0, 1, None, None, None, None, None) == T._lib.EINVAL
    assert lib.tramp_lookup_log_partition(None, None, 1, None, None, None, None, None) == T._lib.EINVAL
    assert lib.tramp_lookup_destroy(None, None) == T._lib.EINVAL
    assert lib.tramp_group_create(None, 1, 1, None, None, 1, C.byref(h)) == T._lib.EINVAL
    assert lib.tramp_group_norm(None, None, None) == T._lib.EINVAL
    assert lib.tramp_group_clip(None, None, 1.0, None, None) == T._lib.EINVAL
    assert lib.tramp_group_limit_step(None, None, None, 1.0, None, 0, 0, None, None, None) == T._lib.EINVAL
    assert lib.tramp_group_destroy(None, None) == T._lib.EINVAL


@pytest.fixture(scope="module")
def buffers(tmp_path_factory):
    "csrc/lookup_buffers.h behind two C functions"
    d = tmp_path_factory.mktemp("buffers")
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    (d / "b.cpp").write_text('#include <initializer_list>\n#include "lookup_buffers.h"\n'
                             'extern "C" const char* conflict(const LkBuffers* m) { return lk_conflict(*m); }\n'
                             'extern "C" int in_place(const void* az, const void* ax, const void* a, const void* v, const void* n) '
                             '{ return lk_scalars_in_place(az, ax, a, v, n); }\n')
    subprocess.run(["g++", "-std=c++17", "-Wall", "-Werror", "-shared", "-fPIC", "-I", os.path.join(root, "tramp_amd", "csrc"), str(d / "b.cpp"),
                    "-o", str(d / "b.so")], check=True)
    lib = C.CDLL(str(d / "b.so"))
    lib.conflict.restype = C.c_char_p
    lib.in_place.argtypes = [C.c_void_p] * 5
    return lib


# 2 instances, z of 2 x 3 doubles, x of 2 x 5, message to x; every buffer on a page of its own
PLACES = dict(az=0x1000, ax=0x2000, a_old=0x3000, bz=0x4000, bx=0x5000, b_old=0x6000, a_new=0x7000, v=0x8000, n_eff=0, b_new=0x9000, r=0xa000)
SIZES = dict(scal=16, nz=48, nx=80, nout=80)


@pytest.mark.parametrize("moved, fine", [
    ({}, True), (dict(a_new=0x3000, b_new=0x6000), True), (dict(a_new=0x1000), True), (dict(v=0x1000), True), (dict(v=0x2000), True),
    (dict(v=0x3000), True), (dict(a_new=0x1000, v=0x2000), True), (dict(a_new=0x1010), True), (dict(r=0), True), (dict(a_new=0x5050), True),
    (dict(a_new=0x1008), False), (dict(a_new=0xff8), False), (dict(v=0x2008), False), (dict(v=0x3008), False), (dict(v=0x7000), False),
    (dict(v=0x7008), False), (dict(a_new=0x4000), False), (dict(a_new=0x5048), False), (dict(v=0x6040), False), (dict(v=0x9000), False),
    (dict(a_new=0xa040), False), (dict(b_new=0x1000), False), (dict(b_new=0x2008), False), (dict(r=0x2000 - 72), False), (dict(r=0x3000), False),
    (dict(b_new=0x5000), False), (dict(b_new=0x4028), False), (dict(b_new=0x6008), False), (dict(r=0x6000), False), (dict(r=0x9008), False),
    (dict(n_eff=0x7008), False), (dict(n_eff=0x1000), True), (dict(n_eff=0x1008), False)])
def test_results_over_what_is_read(buffers, moved, fine):
    fields = ["az", "ax", "a_old", "bz", "bx", "b_old", "a_new", "v", "n_eff", "b_new", "r"]

    class Buffers(C.Structure):
        _fields_ = [(f, C.c_void_p) for f in fields] + [(f, C.c_size_t) for f in ("scal", "nz", "nx", "nout")]
    got = buffers.conflict(C.byref(Buffers(**{**PLACES, **SIZES, **moved})))
    assert (got is None) == fine, got


def test_scalars_over_the_precisions_are_seen(buffers):
    a, b, c, d, e = 0x1000, 0x2000, 0x3000, 0x4000, 0x5000
    assert not buffers.in_place(a, b, c, d, e) and not buffers.in_place(a, b, None, None, None)
    for over in (a, b):
        for results in ((over, d, e), (c, over, e), (c, d, over)):
            assert buffers.in_place(a, b, *results)


def test_instances_by_xcd_stay_within_the_first_axis(tmp_path):
    "fewer than 2^32 work-items along x: an ensemble too large for that goes as (workgroups, instances)"
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    (tmp_path / "g.cpp").write_text('#include "lookup_grid.h"\nextern "C" int spread(size_t batch, size_t blocks) { return lk_spread(batch, blocks, 0, 1); }\n')
    subprocess.run(["g++", "-std=c++17", "-Wall", "-Werror", "-shared", "-fPIC", "-I", os.path.join(root, "tramp_amd", "csrc"),
                    str(tmp_path / "g.cpp"), "-o", str(tmp_path / "g.so")], check=True)
    lib = C.CDLL(str(tmp_path / "g.so"))
    lib.spread.argtypes = [C.c_size_t] * 2
    for batch in (7, 8, 64, 1024, 65528, 65535):
        rounded = (batch + 7) // 8 * 8
        most = (2**32 // 256 - 1) // rounded
        assert rounded * most * 256 < 2**32 <= rounded * (most + 1) * 256
        assert lib.spread(batch, most) and lib.spread(batch, 1) and not lib.spread(batch, most + 1) and not lib.spread(batch, 2**31)
    assert not lib.spread(1, 1) and not lib.spread(9, 1)


def test_iterate_refuses_bad_steps():
    ep = object.__new__(T.ExpectationPropagation)
    ep.default_stopping = T.EarlyStoppingEP()
    for bad in (0, -1.0, np.nan, True, "adaptive", [1.0]):
        with pytest.raises(ValueError):
            ep.iterate(max_step=bad)
    with pytest.raises(ValueError):
        ep.iterate(max_step=1.0, damping="adaptive")


# ---------------------------------------------------------------- the plain definitions against the dense oracle
@pytest.mark.parametrize("V, T_, pad", [(6, 17, 0), (9, 4, 1), (1, 3, 1), (5, 1, 0)])
@pytest.mark.parametrize("scale", [1.0, -2.5])
def test_plain_lookup_is_the_linear_channel_of_its_matrix(V, T_, pad, scale):
    rs = np.random.RandomState(V * T_)
    tok = rs.randint(0, V, T_)
    if pad and T_ > 1:
        tok[1] = -1
    W = dense_of(tok, V, 1, scale)
    lin, lk = orc.LinearOracle(W), LookupFactor(tok, V, 1, scale)
    bz, bx = rs.standard_normal(V), rs.standard_normal(T_)
    for az, ax in [(1.3, 0.7), (0.2, 5.0), (2.0, 0.0), (1e-3, 1e3)]:
        for d in ("forward", "backward"):
            a, b = getattr(lin, d + "_message")(az, bz, ax, bx)
            a2, b2 = getattr(lk, d)(az, bz, ax, bx)
            np.testing.assert_allclose(a2, a, rtol=1e-8, atol=1e-11)
            np.testing.assert_allclose(b2, b, rtol=1e-8, atol=1e-8 * (np.abs(b).max() + 1))
        assert lk.log_partition(az, bz, ax, bx) == pytest.approx(orc.linear_log_partition(lin, az, bz, ax, bx), rel=1e-10)
        assert lk.n_eff(az, ax) == pytest.approx(lin.n_eff(az, ax), rel=1e-10, abs=1e-14)
    assert lk.second_moment(0.7) == pytest.approx(lin.second_moment(0.7), rel=1e-12)


def test_plain_clip_and_step():
    rs = np.random.RandomState(0)
    x = [rs.standard_normal((3, n)) for n in (4, 7)]
    p = [rs.standard_normal((3, n)) for n in (4, 7)]
    norm, y = clip_plain(x, 2.0)
    np.testing.assert_allclose(norm, np.linalg.norm(np.concatenate(x, axis=1), axis=1))
    np.testing.assert_allclose(np.linalg.norm(np.concatenate(y, axis=1), axis=1), np.minimum(norm, 2.0))
    norm, y, c = step_plain(x, p, 1.5)
    np.testing.assert_allclose(np.linalg.norm(np.concatenate(y, axis=1) - np.concatenate(p, axis=1), axis=1), np.minimum(norm, 1.5))
    x[0][1, 2], x[1][2, 0] = np.nan, np.inf
    norm, y = clip_plain(x, 1e-3)
    assert np.isnan(norm[1]) and np.isinf(norm[2])
    for b in (1, 2):
        for u, w in zip(x, y):
            np.testing.assert_array_equal(u[b], w[b])
