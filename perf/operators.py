"""Timed cases of the lookup channel and of the norms over many arrays.

``own`` chooses the side: False computes the operators from elementary operations, True calls
``tramp_amd.LookupChannel`` and ``tramp_amd.ArrayGroup``.  Both sides take the state ``prepare`` makes.

The lookup channel is x[t] = scale * z[token_t] for a table z of V rows and D columns; ``op`` is

  lookup    x from z
  gradient  the adjoint: g[v] = scale * sum of x[t] over the positions t of token v
  backward  the EP message to the table       (a', b')
  forward   the EP message to the positions   (a', b')

and over a list of arrays [instances, n_i]

  clip      every array times min(1, max_norm / norm), the norm taken over all arrays of one instance
  step      previous + min(1, max_norm / norm) * (new - previous), the norm that of new - previous
"""
import math

import numpy as np
import torch

own = False

_TORCH = {"f32": torch.float32, "f64": torch.float64}
_NUMPY = {"f32": np.float32, "f64": np.float64}
_SIZE = {"f32": 4, "f64": 8}
_LOOKUPS = ("lookup", "gradient", "forward", "backward")
_MAX_BYTES = 1.6e9            # what a drawn case may move at most: less than the largest listed one


def _table(name, op, V, T, D, dtype, batch=1, zipf=1.0, pad=0.0):
    return dict(name=name, op=op, V=V, T=T, D=D, dtype=dtype, batch=batch, zipf=zipf, pad=pad)


def _arrays(name, op, k, total, dtype, batch=1, spread=1.0):
    return dict(name=name, op=op, k=k, total=total, dtype=dtype, batch=batch, spread=spread)


def listed():
    return [
        # one position read from a table: a single query of a trained table, all latency
        _table("lookup_one", "lookup", 2000, 1, 64, "f32", zipf=0.0),
        # a ragged batch of sequences, padded: wide rows, most of the traffic the positions written
        _table("lookup_padded_batch", "lookup", 32000, 65536, 1024, "f32", pad=0.2),
        # the adjoint for the same kind of batch: natural (Zipf) frequencies, a few rows collect thousands of positions
        _table("gradient_zipf", "gradient", 32000, 65536, 1024, "f32", pad=0.2),
        # repeated scalar measurements: one column, odd sizes, double precision
        _table("gradient_scalar", "gradient", 100003, 1000001, 1, "f64", zipf=0.8),
        # EP on a small categorical regression: N = 1000 levels, alpha = 2
        _table("backward_small", "backward", 1000, 2000, 1, "f64"),
        # an ensemble of instances over one design, an odd number of columns
        _table("backward_ensemble", "backward", 10007, 80021, 21, "f64", batch=8, zipf=0.7),
        # missing entries: N = 200000 components of which half are observed, once each or so
        _table("forward_observed", "forward", 200000, 100000, 1, "f64", batch=64, zipf=0.0),
        # the large training set: a million rows
        _table("forward_large", "forward", 50000, 1000000, 64, "f32"),
        # the four messages of a GLM chain, N = 1000, M = 500
        _arrays("step_chain_small", "step", 4, 3000, "f64", spread=0.3),
        # the same at N = 100000, M = 50000 and 64 instances
        _arrays("step_chain_ensemble", "step", 4, 300000, "f64", batch=64, spread=0.3),
        # a list of many small and a few large arrays, odd lengths
        _arrays("clip_many", "clip", 41, 5000001, "f32", spread=2.5),
        # the largest: a gigabyte of arrays
        _arrays("clip_large", "clip", 24, 250000000, "f32", spread=1.0),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    while True:
        dtype = rng.choice(["f32", "f64"])
        if rng.random() < 0.65:
            case = dict(op=rng.choice(_LOOKUPS), V=_log_int(rng, 1, 300000), T=_log_int(rng, 1, 1200000),
                        D=_log_int(rng, 1, 1100), dtype=dtype, batch=rng.choice([1, 1, 1, 2, 3, 8, 64]),
                        zipf=round(rng.uniform(0.0, 1.3), 2), pad=rng.choice([0.0, 0.0, 0.05, 0.3]))
        else:
            case = dict(op=rng.choice(["clip", "step"]), k=_log_int(rng, 1, 48), total=_log_int(rng, 48, 200000000),
                        dtype=dtype, batch=rng.choice([1, 1, 1, 2, 5, 64]), spread=round(rng.uniform(0.0, 2.5), 2))
        if work(case)["bytes"] <= _MAX_BYTES and _footprint(case) <= 2 * _MAX_BYTES:
            return case


def _footprint(case):
    e = _SIZE[case["dtype"]] * case["batch"]
    return e * (3 * (case["V"] + case["T"]) * case["D"] if case["op"] in _LOOKUPS else 3 * case["total"])


def _frequencies(case):
    p = np.arange(1, case["V"] + 1, dtype=np.float64) ** -case["zipf"]
    return p / p.sum()


def _lengths(case):
    "lengths of the arrays of one instance: exp(-spread * i) shares, odd where the rounding leaves them so; they sum to the total"
    w = np.exp(-case["spread"] * np.arange(case["k"]) / max(case["k"] / 4, 1))
    n = np.maximum(1, np.floor(w / w.sum() * (case["total"] - case["k"])).astype(np.int64))
    n[0] += case["total"] - n.sum()
    return [int(x) for x in n]


def work(case):
    e = _SIZE[case["dtype"]] * case["batch"]
    if case["op"] in ("clip", "step"):
        n = case["total"]
        return {"bytes": e * n * (2 if case["op"] == "clip" else 3), "flops": case["batch"] * n * (3 if case["op"] == "clip" else 6)}
    V, T, D = case["V"], case["T"], case["D"]
    seen = T * (1.0 - case["pad"])                                             # positions that read a row
    rows = float(-np.expm1(seen * np.log1p(-np.minimum(_frequencies(case), 1 - 1e-12))).sum())   # expected distinct rows
    rows = min(rows, seen)
    moved = {"lookup": rows + T, "gradient": seen + V, "backward": seen + 2 * V, "forward": rows + 2 * T}[case["op"]]
    ops = {"lookup": T, "gradient": seen + V, "backward": seen + 6 * V, "forward": 6 * T}[case["op"]]
    return {"bytes": e * D * moved + 4.0 * T, "flops": case["batch"] * D * ops}


def _inputs(case, seed):
    g = torch.Generator("cuda").manual_seed(seed)
    dt, B = _TORCH[case["dtype"]], case["batch"]

    def normal(*shape):
        return torch.randn(*shape, generator=g, device="cuda", dtype=dt)

    def uniform(*shape):
        return torch.rand(*shape, generator=g, device="cuda", dtype=torch.float64)

    if case["op"] in ("clip", "step"):
        # magnitudes that differ from array to array; some instances are above the bound and some below
        scale = 10.0 ** (-2.0 * uniform(case["k"]))
        level = 0.5 + uniform(B, 1)
        arrays = [(normal(B, n).double() * scale[i] * level).to(dt) for i, n in enumerate(_lengths(case))]
        typical = math.sqrt(float(sum(n * float(s) ** 2 for n, s in zip(_lengths(case), scale))))
        s = dict(arrays=arrays, max_norm=0.9 * typical)
        if case["op"] == "step":
            s["prev"] = [normal(B, n) for n in _lengths(case)]
            s["arrays"] = [p + d for p, d in zip(s["prev"], arrays)]
        return s
    V, T, D = case["V"], case["T"], case["D"]
    order = torch.randperm(V, generator=g, device="cuda")
    cdf = torch.from_numpy(np.cumsum(_frequencies(case))).cuda()
    tokens = order[torch.searchsorted(cdf, uniform(T) * cdf[-1]).clamp_(max=V - 1)]
    if case["pad"]:
        tokens = torch.where(uniform(T) < case["pad"], torch.full_like(tokens, -1), tokens)
    s = dict(tokens=tokens, scale=math.sqrt(D))
    if case["op"] != "gradient":
        s["z"] = normal(B, V, D)
    if case["op"] != "lookup":
        s["x"] = normal(B, T, D)
    if case["op"] in ("forward", "backward"):
        s["az"], s["ax"] = 0.5 + uniform(B), 0.2 + 2.0 * uniform(B)
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    s["case"] = case
    op, B, dt = case["op"], case["batch"], _TORCH[case["dtype"]]
    new = lambda *shape: torch.empty(*shape, device="cuda", dtype=dt)          # noqa: E731  where the results go
    if op in ("clip", "step"):
        s["out"] = [new(*t.shape) for t in s["arrays"]]
        s["norm"] = torch.empty(B, device="cuda", dtype=torch.float64)
    else:
        s["out"] = new(B, case["T"] if op in ("lookup", "forward") else case["V"], case["D"])
        s["a_out"] = torch.empty(B, device="cuda", dtype=torch.float64)
    if not own:
        return s
    import tramp_amd as T
    ctx = T.default_context(0)

    def view(t):
        "the tensor as the framework's device array, [batch, n]"
        return T.DeviceArray(ctx, (t.shape[0], t.numel() // t.shape[0]) if t.dim() > 1 else tuple(t.shape),
                             np.float64 if t.dtype == torch.float64 else np.float32, ptr=t.data_ptr(), owner=False)

    torch.cuda.synchronize()
    if op in ("clip", "step"):
        s["group"] = T.ArrayGroup([view(t) for t in s["arrays"]])
        s["group_out"] = T.ArrayGroup([view(t) for t in s["out"]])
        if op == "step":
            s["group_prev"] = T.ArrayGroup([view(t) for t in s["prev"]])
        s["d_norm"] = view(s["norm"])
        return s
    s["channel"] = T.LookupChannel(s["tokens"].cpu().numpy(), case["V"], dim=case["D"], scale=s["scale"], padding_index=-1,
                                   dtype=_NUMPY[case["dtype"]], ctx=ctx)
    for name in ("z", "x", "az", "ax", "out", "a_out"):
        if name in s:
            s["d_" + name] = view(s[name])
    return s


def run(s):
    return _own(s) if own else _plain(s)


def _own(s):
    op = s["case"]["op"]
    if op == "clip":
        s["group"].clip(s["max_norm"], out=s["group_out"], norm=s["d_norm"])
        return dict(norm=s["norm"], out=s["out"])
    if op == "step":
        s["group"].limit_step(s["group_prev"], s["max_norm"], out=s["group_out"], norm=s["d_norm"])
        return dict(norm=s["norm"], out=s["out"])
    ch = s["channel"]
    if op == "lookup":
        ch.lookup(s["d_z"], out=s["d_out"])
        return s["out"]
    if op == "gradient":
        ch.gradient(s["d_x"], out=s["d_out"])
        return s["out"]
    message = ch.compute_forward_message if op == "forward" else ch.compute_backward_message
    message(s["d_az"], s["d_z"], s["d_ax"], s["d_x"], out_a=s["d_a_out"], out_b=s["d_out"])
    return dict(a=s["a_out"], b=s["out"])


def _token_sums(x, tokens, V):
    "sums of x [B, T, D] over the positions of each token, in 64 bits (a frequent token's sum is long); tokens V are dropped"
    order = torch.argsort(tokens)
    count = torch.bincount(tokens, minlength=V + 1)
    g = torch.stack([torch.segment_reduce(t[order].double(), "sum", lengths=count, unsafe=True) for t in x])
    return g[:, :V], count[:V].double()


def _plain(s):
    case = s["case"]
    op, dt = case["op"], _TORCH[case["dtype"]]
    if op in ("clip", "step"):
        # long sums, and differences of close numbers: in 64 bits
        steps = [x.double() - p for x, p in zip(s["arrays"], s["prev"])] if op == "step" else [t.double() for t in s["arrays"]]
        norm = sum((t * t).sum(1) for t in steps).sqrt()
        c = torch.where(norm > s["max_norm"], s["max_norm"] / norm, torch.ones_like(norm))[:, None]
        out = [(p + c * t).to(dt) for p, t in zip(s["prev"], steps)] if op == "step" else [(c * t).to(dt) for t in steps]
        return dict(norm=norm, out=out)
    V, scale, keep = case["V"], s["scale"], s["tokens"] >= 0
    if op == "lookup":
        return scale * s["z"][:, s["tokens"].clamp(min=0)] * keep.to(dt)[None, :, None]
    g, count = _token_sums(s["x"], torch.where(keep, s["tokens"], V), V)
    g = scale * g
    if op == "gradient":
        return g.to(dt)
    # the message is what is left of the posterior without the neighbour's part, a small difference: in 64 bits
    az, ax, bz = s["az"][:, None, None], s["ax"][:, None, None], s["z"].double()
    likelihood = scale * scale * ax * count[:, None]                                  # [B, V, 1]: what a row learns from its positions
    precision = az + likelihood
    if op == "backward":
        v = (1 / precision).mean(1)
        a = ((likelihood / precision).mean(1) / v).clamp(1e-11, 1e11)                 # = 1 / v - az
        b = (g * (az + a[:, None]) + bz * (a[:, None] - likelihood)) / precision
        return dict(a=a[:, 0], b=b.to(dt))
    share = (keep / precision[:, :, 0][:, s["tokens"].clamp(min=0)])[:, :, None]       # [B, T, 1]: 1 / precision of the row read
    v = scale * scale * share.mean(1)
    a = ((1 - ax * scale * scale * share).mean(1) / v).clamp(1e-11, 1e11)              # = 1 / v - ax
    b = scale * share * (bz + g)[:, s["tokens"].clamp(min=0)] * (ax + a[:, None]) - s["x"]
    return dict(a=a[:, 0], b=b.to(dt))


def exact(case, seed):
    "the definitions in 64 bits on the host"
    s = {k: v.cpu() if isinstance(v, torch.Tensor) else [t.cpu() for t in v] if isinstance(v, list) else v
         for k, v in _inputs(case, seed).items()}
    op, B = case["op"], case["batch"]
    if op in ("clip", "step"):
        square, out = np.zeros(B), []
        for i, t in enumerate(s["arrays"]):
            d = t.numpy().astype(np.float64)
            if op == "step":
                d -= s["prev"][i].numpy()
            square += (d * d).sum(1)
        norm = np.sqrt(square)
        c = np.minimum(1.0, s["max_norm"] / norm)[:, None]
        for i, t in enumerate(s["arrays"]):
            x = t.numpy().astype(np.float64)
            if op == "step":
                p = s["prev"][i].numpy().astype(np.float64)
                out.append(p + c * (x - p))
            else:
                out.append(c * x)
        return dict(norm=norm, out=out)
    V, T, D, scale = case["V"], case["T"], case["D"], s["scale"]
    if B * (V + T) * D > 2e8:
        return None
    tok = s["tokens"].numpy()
    at = np.flatnonzero(tok >= 0)
    tk = tok[at]
    if op == "lookup":
        x = np.zeros((B, T, D))
        x[:, at] = scale * s["z"].numpy()[:, tk].astype(np.float64)
        return x
    # sums over each token's positions: sort the positions by token, sum the runs
    by = at[np.argsort(tk, kind="stable")]
    ids, starts = np.unique(tok[by], return_index=True)
    g = np.zeros((B, V, D))
    count = np.bincount(tk, minlength=V).astype(np.float64)
    for b in range(B):
        if len(ids):
            g[b, ids] = scale * np.add.reduceat(s["x"][b].numpy()[by].astype(np.float64), starts, axis=0)
    if op == "gradient":
        return g
    az, ax = s["az"].numpy()[:, None], s["ax"].numpy()[:, None]
    eig = scale ** 2 * count                                                          # of W^T W, by row
    precision = az + ax * eig
    wide = az.astype(np.longdouble) + ax.astype(np.longdouble) * eig                  # the scalars end in 1 / v - a: wider than 64 bits
    if op == "backward":
        v, a = (1 / wide).mean(1), az
    else:
        v, a = (eig / wide).sum(1) / T, ax
    a_new = np.clip(1 / np.maximum(v, 1e-20) - a[:, 0], 1e-11, 1e11).astype(np.float64)[:, None]
    bz = s["z"].numpy().astype(np.float64)
    if op == "backward":
        # (bz + g) (az + a') / precision - bz without the difference of equal terms of the rows that no position reads
        b = g * ((az + a_new) / precision)[:, :, None] + bz * ((a_new - ax * eig) / precision)[:, :, None]
    else:
        r = (bz + g) * ((ax + a_new) / precision)[:, :, None]
        b = -s["x"].numpy().astype(np.float64)
        b[:, at] += scale * r[:, tk]
    return dict(a=a_new[:, 0], b=b)
