"""The gated block's operators at sizes where their kernels work in other ways: norms of more rows than the caches hold, and losses' gradients whose classes
do not fit into one piece.  Rows (or classes) repeat those of a small matrix, so that definitions in 64 bits stay small."""
import numpy as np
import pytest

from tests import headops as ho
from tests.test_gpu_blocks import PARAMETERS, _parameters, rng

pytestmark = pytest.mark.gpu


class Tiled:
    """A matrix on the device whose rows are those of `few` again and again, rows `gap` elements (NaN) further apart than they are long,
    `shift` elements into its buffer."""

    def __init__(self, few, m, dtype, gap=0, shift=0):
        from tcbnn_amd import head
        from tcbnn_amd.device import DeviceBuffer
        self.n, self.dtype, self.shift, self.size = few.shape[1], dtype, shift, head.ITEMSIZE[dtype]
        self.ld = self.n + gap
        bits = head.encode(np.pad(few.astype(np.float32), ((0, 0), (0, gap)), constant_values=np.nan), dtype)
        self.few = head.decode(bits, dtype).astype(np.float64)[:, :self.n]
        self.count = shift + m * self.ld
        self.buf = DeviceBuffer.from_numpy(np.concatenate([np.zeros(shift, bits.dtype), np.resize(bits, (m, self.ld)).ravel()]))

    def rows(self, first, last):
        from tcbnn_amd.device import DeviceView
        return DeviceView(self.buf.ptr + (self.shift + first * self.ld) * self.size, ((last - first - 1) * self.ld + self.n) * self.size, self.ld, self.buf)

    def bits(self):
        """All of it, gaps too."""
        from tcbnn_amd import head
        return self.buf.to_numpy(head.storage(self.dtype), (self.count,))

    def get(self):
        from tcbnn_amd import head
        wide = head.decode(self.bits()[self.shift:], self.dtype).reshape(-1, self.ld)
        assert np.isnan(wide[:, self.n:]).all(), "a gap between rows was written"
        return wide[:, :self.n]


def _blank(m, n, dtype, gap=0, shift=0):
    return Tiled(np.full((1, n), np.nan), m, dtype, gap, shift)


PERIOD = 61  # (prime to the number of rows that a launch has under way)


# a little more than the caches' bytes: aligned, odd with gaps, in place, narrow
@pytest.mark.parametrize("m,n,dtype,gap,shift,in_place,kind", [(9000, 4096, "bf16", 0, 0, False, "rms"), (9001, 4001, "f16", 3, 1, False, "layer"),
                                                               (9000, 4096, "bf16", 8, 0, True, "layer"), (5003, 4099, "f32", 1, 1, True, "rms"),
                                                               (120000, 301, "bf16", 1, 1, True, "layer")])
def test_norms_past_the_caches(gpu, m, n, dtype, gap, shift, in_place, kind):
    """The same bits as calls on a fifth of the rows, which go through the caches."""
    from tcbnn_amd import head
    r = rng(m, n)
    x, b = (Tiled(r.standard_normal((PERIOD, n)), m, dtype, gap, shift) for _ in range(2))
    s, y, s_part, y_part = (_blank(m, n, dtype, gap, shift) for _ in range(4))
    step = -(-m // 5)
    assert 4 * m * n * x.size > 1 << 28 > 4 * step * n * x.size
    p, _ = _parameters(rng(n), n, kind, kind)

    def run(first, last, s, y):
        layer = head.BlockNormLayerParam("norms", last - first, n, dtype, kind, kind, 0.625)
        layer.initialize(x.rows(first, last), b.rows(first, last), new_stream_gpu=s.rows(first, last), output_gpu=y.rows(first, last), **p)
        layer.forward()
        ho.sync()
        out = [getattr(layer, name).to_numpy(np.float32, (last - first,)) for name in ("after_rstd_gpu", "before_rstd_gpu")]
        layer.release()
        return out

    parts = [run(first, min(m, first + step), s_part, y_part) for first in range(0, m, step)]
    if in_place:
        s, y = x, b
    whole = run(0, m, s, y)
    np.testing.assert_array_equal(s.bits(), s_part.bits())
    np.testing.assert_array_equal(y.bits(), y_part.bits())
    assert np.isfinite(s.get()).all() and np.isfinite(y.get()).all()
    for got, want in zip(whole, zip(*parts)):
        np.testing.assert_array_equal(got, np.concatenate(want))


@pytest.mark.parametrize("m,n,dtype,gap,shift,in_place,kind", [(7000, 4096, "bf16", 0, 0, False, "rms"), (7001, 4001, "f16", 3, 1, False, "layer"),
                                                               (7000, 4096, "bf16", 8, 0, True, "layer"), (3603, 4099, "f32", 1, 1, True, "rms"),
                                                               (90000, 301, "bf16", 1, 1, True, "layer")])
def test_norms_gradients_past_the_caches(gpu, m, n, dtype, gap, shift, in_place, kind):
    """Rows' gradients are the same bits as those of calls on a fifth of the rows, parameters' gradients their sums but for roundings."""
    from tcbnn_amd import head
    r = rng(m, n)
    s, b, dy, ds = (Tiled(r.standard_normal((PERIOD, n)), m, dtype, gap, shift) for _ in range(4))
    dr, db, dr_part, db_part = (_blank(m, n, dtype, gap, shift) for _ in range(4))
    stats = {name: np.resize((1.0 + 0.1 * r.random(PERIOD)).astype(np.float32), m) for name in ("after_rstd", "before_rstd")}
    if kind == "layer":
        stats.update({name: np.resize((0.1 * r.standard_normal(PERIOD)).astype(np.float32), m) for name in ("after_mean", "before_mean")})
    p, counts = _parameters(rng(n), n, kind, kind)
    names = [name for name in PARAMETERS if p[name] is not None]

    def run(first, last, dr, db):
        layer = head.BlockNormLayerParam("norms", last - first, n, dtype, kind, kind, -1.25)
        layer.initialize(s.rows(first, last), b.rows(first, last), new_stream_gpu=s.rows(first, last), **p,
                         **{k + "_gpu": ho.vector(v[first:last]) for k, v in stats.items()})
        grads = {k: ho.empty(n) for k in names}
        layer.initialize_backward(dy.rows(first, last), ds.rows(first, last), dr.rows(first, last), db.rows(first, last),
                                  **{"grad_%s_gpu" % k: v for k, v in grads.items()})
        layer.backward()
        ho.sync()
        layer.release()
        return {k: v.to_numpy(np.float32, (n,)).astype(np.float64) for k, v in grads.items()}

    step = -(-m // 5)
    assert 6 * m * n * s.size > 1 << 28 > 6 * step * n * s.size
    parts = [run(first, min(m, first + step), dr_part, db_part) for first in range(0, m, step)]
    # the four sums' terms, of which a row's repeat, and two of which are in a parameter's gradient at most
    times = np.bincount(np.arange(m) % PERIOD, minlength=PERIOD).astype(np.float64)
    few = {k: v[:PERIOD, None].astype(np.float64) for k, v in stats.items()}
    yh, xh = (np.abs((v.few - few.get(k + "_mean", 0.0)) * few[k + "_rstd"]) for v, k in ((b, "after"), (s, "before")))
    d, dv = np.abs(dr_part.get()[:PERIOD].astype(np.float64)), np.abs(dy.few)
    A, B, C, D = times @ (d * yh), times @ d, times @ (dv * xh), times @ dv
    pa, pb, gate = (np.abs(counts[k]) for k in ("after_gamma", "after_beta", "gate"))
    terms = {"gate": 1.25 * (pa * A + pb * B), "after_gamma": 1.25 * gate * A, "after_beta": 1.25 * gate * B, "before_gamma": C, "before_beta": D}
    if in_place:
        dr, db = dy, b
    whole = run(0, m, dr, db)
    np.testing.assert_array_equal(dr.bits(), dr_part.bits())
    np.testing.assert_array_equal(db.bits(), db_part.bits())
    assert np.isfinite(dr.get()).all() and np.isfinite(db.get()).all()
    for name in names:  # (either side is off by its number of units; d is known as it was rounded)
        ho.check(whole[name], sum(part[name] for part in parts), 1.1 * (1 + ho.U[dtype]) * 2 * (m + 16) * ho.U32 * terms[name], "grad of " + name)


def _exact(few_x, few_w, few_b):
    """Logits of the few rows and classes, and their errors in fp32."""
    k = few_x.shape[1]
    return few_x @ few_w.T + few_b, (k + 1) * ho.U32 * (np.abs(few_x) @ np.abs(few_w).T + np.abs(few_b))


def _loss_layer(m, k, n, dtype, x, w, b, t, g):
    from tcbnn_amd import head
    dx, dw, db = _blank(m, k, dtype, 0, 1), _blank(n, k, dtype, 0, 1), ho.empty(n)
    layer = head.LinearLossLayerParam("loss", m, k, n, dtype).initialize(w.rows(0, n), b, x.rows(0, m), ho.vector(t, np.int32))
    layer.initialize_backward(ho.vector(g), dx.rows(0, m), dw.rows(0, n), db)
    layer.forward()
    layer.backward()
    ho.sync()
    out = layer.download_output(), dx.get().astype(np.float64), dw.get().astype(np.float64), db.to_numpy(np.float32, (n,)).astype(np.float64)
    layer.release()
    return out


# 256 rows have pieces of 262144 classes, 200 of 335360; odd inputs
@pytest.mark.parametrize("m,k,n", [(256, 16, 262144 + 1003), (256, 24, 2 * 262144 + 5), (200, 13, 400003)])
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_loss_gradients_of_few_rows_in_pieces(gpu, m, k, n, dtype):
    """d in two planes, and the inputs' gradient carried from piece to piece."""
    from tcbnn_amd import _lib
    assert _lib.lib.tcbnn_linear_loss_grad_workspace_bytes(m, k, n, _lib.DTYPES[dtype], 0) < 4 * m * n  # (less than both planes of all classes)
    r, u, period = rng(m, k, n), ho.U32, 307
    x, w = Tiled(r.standard_normal((m, k)), m, dtype), Tiled(0.25 + r.standard_normal((period, k)) / 4, n, dtype)
    few_b = r.standard_normal(period).astype(np.float32)
    t = r.integers(0, n, m).astype(np.int32)
    t[::7], t[1], t[2], t[3] = -1, 0, n - 1, n - 2
    g = (0.5 + r.random(m)).astype(np.float32)
    got, dx, dw, db = _loss_layer(m, k, n, dtype, x, w, np.resize(few_b, n), t, g)
    times = np.bincount(np.arange(n) % period, minlength=period).astype(np.float64)
    z, zerr = _exact(x.few, w.few, few_b.astype(np.float64))
    top = z.max(1)
    lse = top + np.log((times * np.exp(z - top[:, None])).sum(1))
    p = np.exp(z - lse[:, None])
    lse_err = 1.1 * ((times * p * (zerr + u * (4 * (top[:, None] - z) + 6))).sum(1) + (n + 8) * u + 4 * u * (np.abs(lse) + np.log(n)))
    ho.check(got["logsumexp"], lse, lse_err, "logsumexp")
    rows, given = np.arange(m), np.where(t >= 0, t, 0)
    at = given % period
    loss = np.where(t >= 0, lse - z[rows, at], 0.0)
    ho.check(got["loss"], loss, lse_err + zerr[rows, at] + 4 * u * (np.abs(top - z[rows, at]) + np.log(n)), "loss")
    # d of a class that is not given, and of the given one; what the products read of them (two planes) is off by `used`
    gg = np.where(t >= 0, g.astype(np.float64), 0.0)
    d, dt = gg[:, None] * p, gg * (p[rows, at] - 1)
    derr = gg[:, None] * p * (1.1 * (zerr + lse_err[:, None] + u * (4 * np.abs(z) + 4 * np.abs(lse)[:, None] + 6)) + u)
    tiny = {"bf16": 2.0 ** -126, "f16": 2.0 ** -38 * gg.max()}[dtype]
    used = derr + ho.U[dtype] ** 2 * (d + derr) + tiny
    used_t = derr[rows, at] + u * np.abs(dt) + ho.U[dtype] ** 2 * np.abs(dt) + tiny
    wt, xa, wa = w.few[at], np.abs(x.few), np.abs(w.few)
    exact = (times * d) @ w.few + (dt - d[rows, at])[:, None] * wt
    err = (times * used) @ wa + used_t[:, None] * np.abs(wt) + (n + 32) * u * 1.01 * ((times * d) @ wa + np.abs(dt)[:, None] * np.abs(wt))
    ho.check(dx, exact, 1.1 * err + ho.U[dtype] * (np.abs(exact) + err) + ho.TINY[dtype], "grad of input")
    exact, err = np.resize(d.T @ x.few, (n, k)), np.resize(used.T @ xa + m * u * 1.01 * (d.T @ xa), (n, k))
    exact_b, err_b = np.resize(d.sum(0), n), np.resize(derr.sum(0) + m * u * 1.01 * d.sum(0), n)
    for i in range(m):  # (the classes that are given, here)
        extra = dt[i] - d[i, at[i]]
        exact[given[i]] += extra * x.few[i]
        err[given[i]] += (used_t[i] + (m + 1) * u * 1.01 * np.abs(dt[i])) * xa[i]
        exact_b[given[i]] += extra
        err_b[given[i]] += used_t[i] + (m + 1) * u * 1.01 * np.abs(dt[i])
    ho.check(dw, exact, 1.1 * err + ho.U[dtype] * (np.abs(exact) + err) + ho.TINY[dtype], "grad of weight")
    ho.check(db, exact_b, 1.1 * err_b + ho.TINY["f32"], "grad of bias")


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_loss_gradients_of_a_last_piece_shorter_than_a_vector(gpu, dtype):
    """Pieces of 256 classes, which is the least, and two classes more; the rows repeat."""
    m, k, n, period, u = 530000, 8, 258, 307, ho.U32
    r = rng(m, k, n)
    x, w = Tiled(r.standard_normal((period, k)), m, dtype), Tiled(0.25 + r.standard_normal((n, k)) / 4, n, dtype)
    b = r.standard_normal(n).astype(np.float32)
    few_t = r.integers(0, n, period).astype(np.int32)
    few_t[::7], few_t[1], few_t[2], few_t[3] = -1, 256, 257, 255
    few_g = (0.5 + r.random(period)).astype(np.float32)
    got, dx, dw, db = _loss_layer(m, k, n, dtype, x, w, b, np.resize(few_t, m), np.resize(few_g, m))
    times = np.bincount(np.arange(m) % period, minlength=period).astype(np.float64)
    z, zerr = _exact(x.few, w.few, b.astype(np.float64))
    top = z.max(1)
    lse = top + np.log(np.exp(z - top[:, None]).sum(1))
    p = np.exp(z - lse[:, None])
    lse_err = 1.1 * ((p * (zerr + u * (4 * (top[:, None] - z) + 6))).sum(1) + (n + 8) * u + 4 * u * (np.abs(lse) + np.log(n)))
    for i in range(0, m, period):  # (every row alike, wherever it lies)
        np.testing.assert_array_equal(got["logsumexp"][i:i + period], got["logsumexp"][:min(period, m - i)])
        np.testing.assert_array_equal(dx[i:i + period], dx[:min(period, m - i)])
    ho.check(got["logsumexp"][:period], lse, lse_err, "logsumexp")
    gg = np.where(few_t >= 0, few_g.astype(np.float64), 0.0)
    one = np.zeros((period, n))
    one[np.arange(period), np.where(few_t >= 0, few_t, 0)] = 1.0
    d = gg[:, None] * (p - one)
    derr = gg[:, None] * (1.1 * p * (zerr + lse_err[:, None] + u * (4 * np.abs(z) + 4 * np.abs(lse)[:, None] + 6)) + u * np.abs(p - one))
    used = derr + ho.U[dtype] * (np.abs(d) + derr) + {"bf16": 2.0 ** -126, "f16": 2.0 ** -38 * gg.max()}[dtype]
    exact, err = d @ w.few, used @ np.abs(w.few) + (n + 32) * u * 1.01 * (np.abs(d) @ np.abs(w.few))
    ho.check(dx[:period], exact, 1.1 * err + ho.U[dtype] * (np.abs(exact) + err) + ho.TINY[dtype], "grad of input")
    xa, dn = np.abs(x.few), times[:, None] * d
    exact, err = dn.T @ x.few, (times[:, None] * used).T @ xa + m * u * 1.01 * (np.abs(dn).T @ xa)
    ho.check(dw, exact, 1.1 * err + ho.U[dtype] * (np.abs(exact) + err) + ho.TINY[dtype], "grad of weight")
    ho.check(db, dn.sum(0), 1.1 * ((times[:, None] * derr).sum(0) + m * u * 1.01 * np.abs(dn).sum(0)) + ho.TINY["f32"], "grad of bias")
