"""Definitions in 64 bits of the lookup channel and of the operators over lists of arrays, with NumPy only; what the tests of
both compare with.  Not collected by pytest."""
from fractions import Fraction

import numpy as np

from oracle import tramp_oracle as orc


def dense_of(tok, V, D, scale):
    "the design matrix [T D, V D]"
    tok = np.asarray(tok).reshape(-1)
    W = np.zeros((tok.size, V))
    at = np.flatnonzero(tok >= 0)
    W[at, tok[at]] = scale
    return np.kron(W, np.eye(D))


class LookupFactor(orc.OracleFactor):
    """x[t] = scale z[tok[t]], tok = -1: padded.  z of V D numbers, x of T D; one instance."""
    kind = "channel"

    def __init__(self, tok, V, D=1, scale=1.0):
        self.tok = np.asarray(tok).reshape(-1)
        self.V, self.D, self.T, self.s = V, D, self.tok.size, scale
        self.at = np.flatnonzero(self.tok >= 0)
        self.count = np.bincount(self.tok[self.at], minlength=V).astype(float)

    def lookup(self, z):
        x = np.zeros((self.T, self.D))
        x[self.at] = self.s * np.asarray(z, dtype=float).reshape(self.V, self.D)[self.tok[self.at]]
        return x

    def gradient(self, x):
        g = np.zeros((self.V, self.D))
        np.add.at(g, self.tok[self.at], np.asarray(x, dtype=float).reshape(self.T, self.D)[self.at])
        return self.s * g

    def _prec(self, az, ax):
        return az + ax * self.s**2 * self.count

    def mean(self, az, bz, ax, bx):
        return (np.asarray(bz, dtype=float).reshape(self.V, self.D) + self.gradient(bx)) / self._prec(az, ax)[:, None]

    def n_eff(self, az, ax):
        if ax == 0:
            return 0.0
        lik = ax * self.s**2 * self.count
        return np.sum(lik[self.count > 0] / (az + lik)[self.count > 0]) / self.V

    def _a(self, v, a):
        "clip(1 / v - a) of a rational v: exact, rounded once"
        return min(max(float(1 / max(v, Fraction(1e-20)) - Fraction(a)), 1e-11), 1e11)

    def _sum(self, az, ax, weight):
        "sum over the rows of weight(count) / (az + ax scale^2 count), exactly"
        count, rows = np.unique(self.count, return_counts=True)
        az, lik = Fraction(az), Fraction(ax) * Fraction(self.s)**2
        return sum((Fraction(int(m)) * weight(Fraction(int(c))) / (az + lik * int(c)) for c, m in zip(count, rows) if weight(c)), Fraction(0))

    def backward_variance(self, az, ax):
        return self._sum(max(az, 1e-11), ax, lambda c: 1) / self.V

    def forward_variance(self, az, ax):
        return Fraction(self.s)**2 * self._sum(az, ax, lambda c: c) / self.T

    def backward(self, az, bz, ax, bx):
        az = max(az, 1e-11)
        a = self._a(self.backward_variance(az, ax), az)
        lik, prec = (ax * self.s**2 * self.count)[:, None], self._prec(az, ax)[:, None]
        b = (self.gradient(bx) * (az + a) + np.asarray(bz, dtype=float).reshape(self.V, self.D) * (a - lik)) / prec
        return a, b.reshape(np.shape(bz))

    def forward(self, az, bz, ax, bx):
        a = self._a(self.forward_variance(az, ax), ax)
        rx = np.zeros((self.T, self.D))
        rx[self.at] = self.s * self.mean(az, bz, ax, bx)[self.tok[self.at]]
        return a, rx.reshape(np.shape(bx)) * (ax + a) - np.asarray(bx, dtype=float)

    def log_partition(self, az, bz, ax, bx):
        prec = self._prec(az, ax)
        h = np.asarray(bz, dtype=float).reshape(self.V, self.D) + self.gradient(bx)
        return 0.5 * np.sum(h**2 / prec[:, None]) + 0.5 * self.D * np.sum(np.log(2 * np.pi / prec))

    def second_moment(self, tau_z):
        return tau_z * self.s**2 * self.at.size / self.T


def _factor(norm, bound):
    with np.errstate(all="ignore"):
        return np.where(np.isfinite(norm) & (norm > bound), bound / norm, 1.0)


def _norm(arrays):
    return np.sqrt(sum((np.asarray(x, dtype=float)**2).sum(axis=1) for x in arrays))


def clip_plain(arrays, bound):
    norm = _norm(arrays)
    c = _factor(norm, bound)[:, None]
    return norm, [np.where(c < 1, c * np.asarray(x, dtype=float), x) for x in arrays]


def step_plain(arrays, prev, bound):
    with np.errstate(all="ignore"):
        d = [np.asarray(x, dtype=float) - np.asarray(p, dtype=float) for x, p in zip(arrays, prev)]
        norm = _norm(d)
        c = _factor(norm, bound)[:, None]
        return norm, [np.where(c < 1, np.asarray(p, dtype=float) + c * t, x) for x, p, t in zip(arrays, prev, d)], c[:, 0]


def zipf_tokens(rs, V, T, exponent=1.0, pad=0.0):
    p = np.arange(1, V + 1, dtype=float)**-exponent
    tok = rs.permutation(V)[rs.choice(V, size=T, p=p / p.sum())]
    tok[rs.uniform(size=T) < pad] = -1
    return tok
