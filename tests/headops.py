"""numpy wrappers that run the float head's layers, their definitions in 64 bits, and the error that a kernel may have
(test helper).

Tolerances follow from the arithmetic: a sum of n fp32 terms, in any order, is off by at most n u32 sum |terms|; an output
is rounded once to its type (u below); what is rounded on the way (dz in 16-bit types) adds u of its terms."""
import numpy as np
from scipy.special import erf

from tcbnn_amd import _lib, head
from tcbnn_amd.device import DeviceBuffer, DeviceView

U32 = 2.0 ** -24
U = {"f32": 2.0 ** -24, "bf16": 2.0 ** -8, "f16": 2.0 ** -11}  # half the distance of neighbours, relative
TINY = {"f32": 2.0 ** -126, "bf16": 2.0 ** -126, "f16": 2.0 ** -25}  # results below the normal numbers
DTYPES = ["f32", "bf16", "f16"]


def rounded(x, dtype):
    """(bits, the fp64 values they stand for)"""
    bits = head.encode(x, dtype)
    return bits, head.decode(bits, dtype).astype(np.float64)


class Matrix:
    """A matrix on the device, rows `gap` elements further apart than they are long, every gap element NaN.  It begins `shift`
    elements into its buffer: with one, rows of odd length start at every alignment there is; with none, rows whose length
    and gap are multiples of 16 bytes lie at whole 16 bytes."""

    def __init__(self, values, dtype, gap=0, rows=None, cols=None, shift=1):
        if values is None:  # an output: NaN everywhere
            values = np.full((rows, cols), np.nan, np.float32)
        self.shape, self.dtype, self.gap, self.shift = values.shape, dtype, gap, shift
        wide = np.full((values.shape[0], values.shape[1] + gap), np.nan, np.float32)
        wide[:, :values.shape[1]] = values
        bits = head.encode(wide, dtype)
        self.values = head.decode(bits, dtype).astype(np.float64)[:, :values.shape[1]]
        self.buf = DeviceBuffer.from_numpy(np.concatenate([np.zeros(shift, bits.dtype), bits.ravel()]))
        self.view = DeviceView(self.buf.ptr + shift * bits.itemsize, bits.nbytes, wide.shape[1] if gap else 0, self.buf)

    def get(self):
        wide = self.buf.to_numpy(head.storage(self.dtype), (self.shift + self.shape[0] * (self.shape[1] + self.gap),))[self.shift:]
        wide = head.decode(wide, self.dtype).reshape(self.shape[0], -1)
        assert np.isnan(wide[:, self.shape[1]:]).all(), "a gap between rows was written"
        return wide[:, :self.shape[1]].astype(np.float64)


def vector(values, dtype=np.float32):
    return DeviceBuffer.from_numpy(np.asarray(values, dtype))


def empty(n, dtype=np.float32):
    return DeviceBuffer.from_numpy(np.full(n, 0x7f7f7f7f, np.uint32).view(dtype))


def sync():
    _lib.device_synchronize()


def check(got, want, tol, what=""):
    got, want = np.asarray(got, np.float64), np.asarray(want, np.float64)
    assert got.shape == want.shape, (what, got.shape, want.shape)
    special = ~np.isfinite(want)
    np.testing.assert_array_equal(got[special], want[special], err_msg=what)
    err = np.abs(got[~special] - want[~special])
    bad = ~(err <= np.broadcast_to(tol, want.shape)[~special])
    assert not bad.any(), "%s: %d of %d off, by up to %g (allowed there %g)" % (
        what, bad.sum(), bad.size, err[bad].max(), np.broadcast_to(tol, want.shape)[~special][bad][err[bad].argmax()])


# ---- definitions in 64 bits
def act(name, z):
    if name == "relu":
        return np.maximum(z, 0)
    if name == "gelu":
        return 0.5 * z * (1 + erf(z / np.sqrt(2)))
    if name == "silu":
        return z / (1 + np.exp(-z))
    return z


def slope(name, z):
    if name == "relu":
        return (z > 0).astype(np.float64)
    if name == "gelu":
        return 0.5 * (1 + erf(z / np.sqrt(2))) + z * np.exp(-0.5 * z * z) / np.sqrt(2 * np.pi)
    if name == "silu":
        p = 1 / (1 + np.exp(-z))
        return p * (1 + z * (1 - p))
    return np.ones_like(z)


def norm(x, gamma, beta, eps):
    mean = x.mean(1, keepdims=True)
    rstd = 1 / np.sqrt(((x - mean) ** 2).mean(1, keepdims=True) + eps)
    return (x - mean) * rstd * gamma + beta, mean[:, 0], rstd[:, 0]


def order(x):
    """Classes of a row, best first: NaN, then larger values; lower indices among equals."""
    key = np.where(np.isnan(x), np.inf, x)
    return np.lexsort((np.arange(len(x)), -key, ~np.isnan(x)))


def logprobs(x, t, top):
    """One row: logprob, entropy, logsumexp, rank, top_index, top_logprob."""
    n = len(x)
    with np.errstate(invalid="ignore", divide="ignore", over="ignore"):
        m = x.max()
        if m == -np.inf:
            lse, entropy, lp = -np.inf, 0.0, np.full(n, -np.inf)
        else:
            lse = m + np.log(np.exp(x - m).sum())
            lp = x - lse if np.isfinite(m) else np.full(n, np.nan)
            p = np.exp(lp)
            entropy = -(p * np.where(p > 0, lp, 0)).sum() if np.isfinite(m) else np.nan
            lse = lse if np.isfinite(m) else np.nan
    best = order(x)
    logprob = 0.0 if t < 0 else (lp[t] if t < n else np.nan)
    rank = int(np.nonzero(best == t)[0][0]) if 0 <= t < n else -1
    return logprob, entropy, lse, rank, best[:top], lp[best[:top]]
