"""The linear loss where logits are far from 0: finite masks of every size over whole tiles and over a wavefront's columns, and rows all of whose
logits are there.  Inputs are whole numbers, so that logits are known to the bit."""
import numpy as np
import pytest

from tests import blockops as bo
from tests import headops as ho
from tests.test_gpu_blocks import _loss, rng

pytestmark = pytest.mark.gpu

MASKS = [-1e5, -1e9, -1e10, -1e20, -1e30, -8e37]
# few rows, one row that takes tiles, and every tile: 32, 64, 128, 128 deep, 128 with one step in LDS, 256; rows that lie anywhere
SIZES = [(1, 64, 200, 0), (1, 2048, 8192, 0), (12, 40, 700, 1), (33, 72, 300, 0), (100, 61, 304, 1), (1024, 72, 1500, 0), (1000, 71, 1500, 1), (2040, 72, 2052, 0),
         (2040, 72, 2052, 1), (2048, 64, 2048, 0), (2048, 64, 3100, 0)]


def _masked(gpu, m, k, n, dtype, shift, mask, want=()):
    allowed = n - n // 2
    t = rng(m, n).integers(-1, allowed, m).astype(np.int32)
    _loss(gpu, m, k, n, dtype, shift=shift, forbidden=np.arange(allowed, n), t=t, mask=mask, want=want)
    # one wavefront's 32 or 64 columns, with classes on both sides
    first = n // 2 // 64 * 64
    t[t >= first] -= first
    _loss(gpu, m, k, n, dtype, shift=shift, forbidden=np.arange(first, min(n, first + 64)), t=t, mask=mask, want=want)


@pytest.mark.parametrize("dtype", ho.DTYPES)
@pytest.mark.parametrize("m,k,n,shift", SIZES)
def test_loss_of_classes_masked_by_any_value(gpu, m, k, n, shift, dtype):
    for mask in MASKS if m * n < 1 << 20 else [-1e10, -1e30]:
        _masked(gpu, m, k, n, dtype, shift, mask)
    _masked(gpu, m, k, n, dtype, shift, -1e20, ("input", "weight", "bias"))


@pytest.mark.parametrize("m,k,n,dtype", [(1500, 520, 6000, "bf16"), (4096, 256, 4096, "f32")])
def test_loss_of_masked_classes_in_the_largest_tiles(gpu, m, k, n, dtype):
    _masked(gpu, m, k, n, dtype, 0, -1e10)


def _whole(r, rows, k, dtype, shift):
    """A matrix of -1, 0 and 1, of which any product is exact."""
    return ho.Matrix(r.integers(-1, 2, (rows, k)).astype(np.float64), dtype, shift=shift)


def _logits(x, w, b):
    """As fp32 holds them: the products are whole numbers, the bias is added once."""
    return ((x.values @ w.values.T).astype(np.float32) + b[None, :]).astype(np.float64)


# what all logits of a row are about
FAR = [3e4, -3e4, 1e6, -1e6, 1e9, -1e9, 1e10, -1e10, 1e12, 1e20, -1e20, -1e30, 1e37, -8e37]


@pytest.mark.parametrize("dtype", ho.DTYPES)
@pytest.mark.parametrize("m,k,n,shift", SIZES)
def test_loss_of_rows_all_far_from_0(gpu, m, k, n, shift, dtype):
    from tcbnn_amd import head
    r = rng(m, k, n)
    x, w = _whole(r, m, k, dtype, shift), _whole(r, n, k, dtype, shift)
    t = r.integers(0, n, m).astype(np.int32)
    for value in FAR if m * n < 1 << 20 else FAR[::3]:
        b = np.full(n, value, np.float32)
        layer = head.LinearLossLayerParam("loss", m, k, n, dtype).initialize(w.view, b, x.view, ho.vector(t, np.int32))
        layer.forward()
        ho.sync()
        z = _logits(x, w, b)
        top = z.max(1, keepdims=True)
        e = np.exp(z - top)
        s = e.sum(1)
        lse, loss = top[:, 0] + np.log(s), top[:, 0] - z[np.arange(m), t] + np.log(s)
        # exp's argument, exp by some units and the sum of n; the logarithm of it, and one rounding of each difference
        err = (e / s[:, None] * (4 * (top - z) + 6)).sum(1) + n + 8 + 4 * np.log(n + 1.0)
        got = layer.download_output()
        ho.check(got["logsumexp"], lse, 1.1 * ho.U32 * (err + 2 * np.abs(lse)), "logsumexp at %g" % value)
        ho.check(got["loss"], loss, 1.1 * ho.U32 * (err + 4 * np.abs(loss)), "loss at %g" % value)
        layer.release()


@pytest.mark.parametrize("dtype", ho.DTYPES)
@pytest.mark.parametrize("m,k,n,shift", [(1, 64, 200, 0), (3, 24, 70, 1), (12, 40, 700, 1), (40, 72, 300, 0), (300, 61, 304, 1), (1024, 72, 1500, 0), (2040, 72, 2052, 0),
                                         (2048, 64, 3100, 0)])
def test_loss_gradient_of_a_certain_class_far_from_0(gpu, m, k, n, shift, dtype):
    """One class of every row is alone at `value`: its p is 1, the others' 0, whatever logsumexp's size."""
    from tcbnn_amd import head
    r = rng(m, k, n)
    x, w = _whole(r, m, k, dtype, shift), _whole(r, n, k, dtype, shift)
    t = r.integers(-1, n, m).astype(np.int32)
    t[0], best = n - 1, n // 3
    if m > 2:
        t[2] = best
    g = (0.5 + r.random(m)).astype(np.float32)
    for value in [1e5, -1e5, 3e9, -3e9, 1e10, -1e10, 1e12, -1e12, 1e20, -1e30, 1e37, -8e37]:
        b = np.full(n, 0.0 if value > 0 else 4 * value, np.float32)
        b[best] = value
        dx, dw, db = ho.Matrix(None, dtype, 0, m, k, shift=0), ho.Matrix(None, dtype, 0, n, k, shift=0), ho.empty(n)
        layer = head.LinearLossLayerParam("loss", m, k, n, dtype).initialize(w.view, b, x.view, ho.vector(t, np.int32))
        layer.initialize_backward(ho.vector(g), dx.view, dw.view, db)
        layer.forward()
        layer.backward()
        ho.sync()
        z = _logits(x, w, b)
        p = np.zeros((m, n))
        p[:, best] = 1.0
        # (p is that of logits about logsumexp: exp's argument is 0, and off by less than 65536 2^-23 where it is that of a rounded product)
        near = np.where(np.abs(z[:, best]) > 65536.0, 0.0, ho.U32 * 2 * 65536)
        exact = bo.loss_grads(x.values, w.values, t, g.astype(np.float64), z - z[:, best:best + 1], 0.0, p, np.zeros(m), near, dtype)
        for name, buf in (("input", dx), ("weight", dw)):
            e, err = exact[name]
            ho.check(buf.get(), e, bo.out_error(e, err, dtype), "grad of %s at %g" % (name, value))
        e, err = exact["bias"]
        ho.check(db.to_numpy(np.float32, (n,)), e, 1.1 * err + ho.TINY["f32"], "grad of bias at %g" % value)
        layer.release()


@pytest.mark.parametrize("dtype", ho.DTYPES)
@pytest.mark.parametrize("m,k,n,shift", [(1, 64, 200, 0), (3, 24, 70, 1), (12, 40, 700, 1), (40, 72, 300, 0), (300, 61, 304, 1), (1024, 72, 1500, 0), (2040, 72, 2052, 0),
                                         (2048, 64, 3100, 0)])
def test_loss_gradients_of_rows_all_far_from_0(gpu, m, k, n, shift, dtype):
    """A row whose mask, or whose size, leaves no class near 0: classes share p as their differences say."""
    from tcbnn_amd import head
    r = rng(m, k, n, 2)
    x, w = _whole(r, m, k, dtype, shift), _whole(r, n, k, dtype, shift)
    t = r.integers(-1, n, m).astype(np.int32)
    g = (0.5 + r.random(m)).astype(np.float32)
    for value in [0.0, *FAR, np.finfo(np.float32).min] if m * n < 1 << 20 else [3e4, -1e6, 1e9, -1e30]:
        b = np.full(n, value, np.float32)
        dx, dw, db = ho.Matrix(None, dtype, 0, m, k, shift=0), ho.Matrix(None, dtype, 0, n, k, shift=0), ho.empty(n)
        layer = head.LinearLossLayerParam("loss", m, k, n, dtype).initialize(w.view, b, x.view, ho.vector(t, np.int32))
        layer.initialize_backward(ho.vector(g), dx.view, dw.view, db)
        layer.forward()
        layer.backward()
        ho.sync()
        z = _logits(x, w, b)
        top = z.max(1, keepdims=True)
        z = z - top
        e = np.exp(z)
        s = e.sum(1)
        p, lse = e / s[:, None], np.log(s)
        lse_err = 1.1 * ho.U32 * ((p * (4 * np.abs(z) + 6)).sum(1) + n + 8 + 4 * np.log(n + 1.0))
        whole, rest = layer.logsumexp_gpu.to_numpy(np.float32, (m,)).astype(np.float64), layer.logsumexp_rest_gpu.to_numpy(np.float32, (m,))
        ho.check(whole - top[:, 0] + rest, lse, lse_err + ho.U32 * np.abs(rest), "logsumexp and its rest at %g" % value)
        exact = bo.loss_grads(x.values, w.values, t, g.astype(np.float64), z, 0.0, p, lse, lse_err, dtype)
        for name, buf in (("input", dx), ("weight", dw)):
            e, err = exact[name]
            ho.check(buf.get(), e, bo.out_error(e, err, dtype), "grad of %s at %g" % (name, value))
        e, err = exact["bias"]
        ho.check(db.to_numpy(np.float32, (n,)), e, 1.1 * err + ho.TINY["f32"], "grad of bias at %g" % value)
        layer.release()


# (one row of the first takes tiles forward and the kernel for few rows backward)
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("m,k,n", [(1, 2048, 8192), (4, 2048, 8192), (12, 4096, 640), (40, 2048, 300), (300, 1000, 777)])
def test_loss_gradients_of_logits_that_are_known_to_no_unit(gpu, m, k, n, dtype):
    """Sums so large that their rounding in another order is many units: p is still no more than 1."""
    from tcbnn_amd import head
    r = rng(m, k, n, 3)
    x, w = (ho.Matrix(3e4 * r.standard_normal((rows, k)), dtype, shift=0) for rows in (m, n))
    g = (0.5 + r.random(m)).astype(np.float32)
    for sign in (1, -1):
        dx, dw, db = ho.Matrix(None, dtype, 0, m, k, shift=0), ho.Matrix(None, dtype, 0, n, k, shift=0), ho.empty(n)
        b = np.full(n, 4e11 * sign, np.float32)
        layer = head.LinearLossLayerParam("loss", m, k, n, dtype).initialize(w.view, b, x.view, ho.vector(r.integers(-1, n, m), np.int32))
        layer.initialize_backward(ho.vector(g), dx.view, dw.view, db)
        layer.forward()
        layer.backward()
        ho.sync()
        out = layer.download_output()
        assert np.isfinite(out["loss"]).all() and np.isfinite(out["logsumexp"]).all()
        # |d| is |g| at most, but for roundings of the loss' exponential and of the sums
        limit = (1 + 2.0 ** -7) * g.sum()
        assert (np.abs(db.to_numpy(np.float32, (n,))) <= limit).all()
        assert (np.abs(dw.get()) <= limit * np.abs(x.values).max()).all()
        # (a class that has the largest logit, and the given one)
        assert np.isfinite(dx.get()).all()
        layer.release()


@pytest.mark.parametrize("dtype", ho.DTYPES)
@pytest.mark.parametrize("m,k,n", [(2, 64, 300), (12, 40, 700), (300, 61, 304)])
def test_loss_without_what_may_be_missing(gpu, m, k, n, dtype):
    """Each output of the forward call alone; gradients from logsumexp alone."""
    from tcbnn_amd import head
    r = rng(m, k, n, 5)
    x, w = (ho.Matrix(r.standard_normal((rows, k)), dtype) for rows in (m, n))
    t, g = r.integers(-1, n, m).astype(np.int32), (0.5 + r.random(m)).astype(np.float32)
    b = (30 + r.standard_normal(n)).astype(np.float32)
    dx, dw, db = ho.Matrix(None, dtype, 0, m, k), ho.Matrix(None, dtype, 0, n, k), ho.empty(n)
    layer = head.LinearLossLayerParam("loss", m, k, n, dtype).initialize(w.view, b, x.view, ho.vector(t, np.int32))
    layer.initialize_backward(ho.vector(g), dx.view, dw.view, db)
    layer.forward()
    names = ("loss", "logsumexp", "logsumexp_rest")
    buffers = [getattr(layer, name + "_gpu") for name in names]
    all_at_once = [buf.to_numpy(np.float32, (m,)) for buf in buffers]
    for i, name in enumerate(names):
        for other in names:
            setattr(layer._desc, other, None)
        alone = ho.empty(m)
        setattr(layer._desc, name, alone.ptr)
        layer._desc.targets = layer.targets_gpu.ptr if name == "loss" else None
        layer.forward()
        ho.sync()
        np.testing.assert_array_equal(alone.to_numpy(np.float32, (m,)), all_at_once[i])
    layer._grad_desc.loss = layer._grad_desc.logsumexp_rest = None
    layer.backward()
    ho.sync()
    _, _, lse, lse_err, z, zerr, p = bo.loss(x.values, w.values, b.astype(np.float64), t, g)
    exact = bo.loss_grads(x.values, w.values, t, g.astype(np.float64), z, zerr, p, lse, lse_err, dtype)
    for name, buf in (("input", dx), ("weight", dw)):
        e, err = exact[name]
        ho.check(buf.get(), e, bo.out_error(e, err, dtype), "grad of " + name)
    e, err = exact["bias"]
    ho.check(db.to_numpy(np.float32, (n,)), e, 1.1 * err + ho.TINY["f32"], "grad of bias")
    layer.release()
