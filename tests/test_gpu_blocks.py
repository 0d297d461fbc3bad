"""The gated block's operators on the GPU against definitions in 64 bits: the norms after and before a block, the gated product, the
loss of a linear classifier, and their gradients; sizes around those where the kernels change, odd sizes, strides, buffers over one another, empty and degenerate
inputs."""
import numpy as np
import pytest

from tests import blockops as bo
from tests import headops as ho

pytestmark = pytest.mark.gpu

GAPS = {"f32": 1, "bf16": 3, "f16": 5}
PARAMETERS = ("gate", "after_gamma", "after_beta", "before_gamma", "before_beta")


def rng(*seed):
    return np.random.default_rng([abs(int(s)) for s in seed])


# --------------------------------------------------------------------------- norms after and before a block
def _parameters(r, n, after, before, gate=True):
    """{name: fp32 vector or None}, {name: what it counts as}"""
    there = {"gate": gate, "after_gamma": after != "none", "after_beta": after == "layer", "before_gamma": before != "none",
             "before_beta": before == "layer"}
    p = {k: (1 if "beta" not in k else 0) + 0.3 * r.standard_normal(n) if there[k] else None for k in PARAMETERS}
    p = {k: None if v is None else v.astype(np.float32) for k, v in p.items()}
    return p, {k: (np.zeros(n) if "beta" in k else np.ones(n)) if v is None else v.astype(np.float64) for k, v in p.items()}


def _norms(gpu, m, n, dtype, after, before, block=True, gate=True, gap=0, in_place=False, stream=None, shift=1, scale=0.625, eps=1e-5,
           values=None):
    from tcbnn_amd import head
    r = rng(m, n, len(dtype), len(after), len(before))
    x = ho.Matrix(2 * r.standard_normal((m, n)) + 0.2 if values is None else values, dtype, gap, shift=shift)
    b = ho.Matrix(1.5 * r.standard_normal((m, n)) + 0.3, dtype, gap, shift=shift) if block else None
    p, counts = _parameters(r, n, after, before, gate and block)
    xv, bv = x.values.copy(), b.values.copy() if block else None
    s = x if in_place else ho.Matrix(None, dtype, gap, m, n) if block else None
    y = (b if in_place and block else ho.Matrix(None, dtype, gap, m, n)) if before != "none" else None
    layer = head.BlockNormLayerParam("norms", m, n, dtype, after, before, scale, eps)
    layer.initialize(x.view, b.view if block else None, new_stream_gpu=s.view if s else None, output_gpu=y.view if y else None, **p)
    layer.forward(stream)
    ho.sync()
    want, err, wy, yerr, first, second = bo.norms(xv, bv, *(counts[k] for k in PARAMETERS), after, before, np.float32(scale).item(),
                                                  np.float32(eps).item())
    if s and block:
        ho.check(s.get(), want, bo.out_error(want, err, dtype), "stream")
    if y:
        ho.check(y.get(), wy, bo.out_error(wy, yerr, dtype), "output")
    for norm, name in ((first, "after"), (second, "before")):
        if norm is None or norm.kind == "none":
            continue
        ho.check(getattr(layer, name + "_rstd_gpu").to_numpy(np.float32, (m,)), norm.rstd, norm.rstd_err + ho.U32 * norm.rstd, name + " rstd")
        if norm.kind == "layer":
            ho.check(getattr(layer, name + "_mean_gpu").to_numpy(np.float32, (m,)), norm.mean, norm.mean_err + ho.U32 * np.abs(norm.mean), name + " mean")
    layer.release()


# one value; a vector of 16 bytes and one to each side; every team of wavefronts, whole and ragged, and beyond registers; more rows than
# workgroups have teams
ROWS = [(1, 1), (1, 7), (2, 8), (3, 64), (4, 255), (5, 513), (9, 1000), (33, 1024), (300, 264), (2, 2048), (7, 4096), (3, 4100), (17, 8192), (2, 8200),
        (3, 16384), (2, 16392), (1, 65536), (3, 40001), (700, 40), (9000, 24), (1100, 2056)]


@pytest.mark.parametrize("dtype", ho.DTYPES)
@pytest.mark.parametrize("m,n", ROWS)
def test_norms(gpu, m, n, dtype):
    for after, before in (("rms", "rms"), [("layer", "layer"), ("none", "layer"), ("layer", "rms"), ("none", "rms")][(m + n) % 4]):
        _norms(gpu, m, n, dtype, after, before)


@pytest.mark.parametrize("after", bo.KINDS)
@pytest.mark.parametrize("before", bo.KINDS)
@pytest.mark.parametrize("m,n", [(5, 40), (35, 1030), (2, 20000)])
def test_norms_of_every_kind(gpu, m, n, after, before):
    for dtype in ho.DTYPES:
        _norms(gpu, m, n, dtype, after, before, gate=False)
        _norms(gpu, m, n, dtype, after, before, gap=GAPS[dtype])
        _norms(gpu, m, n, dtype, after, before, gap=8, shift=0, in_place=True)
        if after == "none" and before != "none":
            _norms(gpu, m, n, dtype, after, before, block=False)


def test_norms_of_degenerate_rows(gpu):
    """Rows of zeros, rows of one value, a row far from zero."""
    for dtype in ho.DTYPES:
        for before in ("rms", "layer"):
            for n in (24, 1000, 33000):
                v = np.zeros((4, n))
                v[1], v[2], v[3, ::2] = 3, -0.5, 1024
                _norms(gpu, 4, n, dtype, "none", before, block=False, values=v)


def test_norms_rows_do_not_mix(gpu):
    from tcbnn_amd import head
    for n in (40, 5000, 30000):
        r = rng(n)
        x, b = r.standard_normal((5, n)), r.standard_normal((5, n))
        x[1, n - 1], b[3, 0] = np.nan, np.inf
        x, b, s, y = ho.Matrix(x, "bf16"), ho.Matrix(b, "bf16"), ho.Matrix(None, "bf16", 0, 5, n), ho.Matrix(None, "bf16", 0, 5, n)
        head.BlockNormLayerParam("norms", 5, n, "bf16", "layer", "rms").initialize(x.view, b.view, new_stream_gpu=s.view, output_gpu=y.view).forward()
        ho.sync()
        np.testing.assert_array_equal(np.isfinite(y.get()).all(1), [True, False, True, False, True])
        np.testing.assert_array_equal(np.isnan(y.get()).all(1), [False, True, False, True, False])


def _norms_grad(gpu, m, n, dtype, after, before, block=True, gate=True, dy=True, ds=True, gap=0, in_place=False, want=None, shift=1, scale=-1.25,
                stream=None):
    from tcbnn_amd import head
    r = rng(m, n, len(dtype), len(after), len(before), 1)
    s = ho.Matrix(2 * r.standard_normal((m, n)) + 0.2, dtype, gap, shift=shift)
    b = ho.Matrix(1.5 * r.standard_normal((m, n)) + 0.3, dtype, gap, shift=shift) if block else None
    p, counts = _parameters(r, n, after, before, gate and block)
    dy = ho.Matrix(r.standard_normal((m, n)), dtype, gap, shift=shift) if dy and before != "none" else None
    ds = ho.Matrix(r.standard_normal((m, n)), dtype, gap, shift=shift) if ds else None
    stats = {}
    for name, x, kind in (("after", b, after), ("before", s, before)):
        if kind == "none" or x is None:
            continue
        mean = x.values.mean(1) if kind == "layer" else np.zeros(m)
        stats[name + "_rstd"] = (1 / np.sqrt(((x.values - mean[:, None]) ** 2).mean(1) + 1e-5)).astype(np.float32)
        stats[name + "_mean"] = mean.astype(np.float32)
    layer = head.BlockNormLayerParam("norms", m, n, dtype, after, before, scale)
    layer.initialize(s.view, b.view if block else None, new_stream_gpu=s.view, **p,
                     **{k + "_gpu": ho.vector(v) for k, v in stats.items() if "rstd" in k or (after if k[0] == "a" else before) == "layer"})
    exact = bo.norms_grad(s.values, b.values if block else None, *(counts[k] for k in PARAMETERS[:4]),
                          {k: v.astype(np.float64) for k, v in stats.items()}, dy and dy.values, ds and ds.values, after, before, scale)
    names = [k for k in PARAMETERS if p[k] is not None and k in exact] if want is None else [k for k in want if k in PARAMETERS]
    grads = {k: ho.empty(n) for k in names}
    dr, db = (ho.Matrix(None, dtype, gap, m, n) if want is None or k in want else None for k in ("stream", "block"))
    if not block:
        db = None
    if in_place:
        dr = ds if ds else dy
        db = dy if block and ds and dy else b if block else None
    layer.initialize_backward(dy.view if dy else None, ds.view if ds else None, dr.view if dr else None, db.view if db else None,
                              **{"grad_%s_gpu" % k: v for k, v in grads.items()})
    layer.backward(stream)
    ho.sync()
    for k, buf in (("stream", dr), ("block", db)):
        if buf:
            g, err = exact[k]
            ho.check(buf.get(), g, bo.out_error(g, err, dtype), "grad of the " + k)
    for k, buf in grads.items():
        g, err = exact[k]
        ho.check(buf.to_numpy(np.float32, (n,)), g, 1.1 * err + ho.U32 * np.abs(g) + ho.TINY["f32"], "grad of " + k)
    layer.release()


@pytest.mark.parametrize("dtype", ho.DTYPES)
@pytest.mark.parametrize("m,n", ROWS)
def test_norms_grad(gpu, m, n, dtype):
    for after, before in (("rms", "rms"), [("layer", "layer"), ("none", "layer"), ("layer", "rms"), ("none", "rms")][(m + n) % 4]):
        _norms_grad(gpu, m, n, dtype, after, before)


@pytest.mark.parametrize("after", bo.KINDS)
@pytest.mark.parametrize("before", bo.KINDS)
@pytest.mark.parametrize("m,n", [(5, 40), (300, 264), (35, 1030), (2, 20000)])
def test_norms_grad_of_every_kind(gpu, m, n, after, before):
    for dtype in ho.DTYPES:
        _norms_grad(gpu, m, n, dtype, after, before, gate=False, gap=GAPS[dtype])
        _norms_grad(gpu, m, n, dtype, after, before, gap=8, shift=0, in_place=True)
        _norms_grad(gpu, m, n, dtype, after, before, ds=before == "none")
        _norms_grad(gpu, m, n, dtype, after, before, dy=False)
        for want in (("stream",), ("block",), ("gate",), ("gate", "block")):
            _norms_grad(gpu, m, n, dtype, after, before, want=want)
        if after == "none" and before != "none":
            _norms_grad(gpu, m, n, dtype, after, before, block=False)
        if before != "none":
            _norms_grad(gpu, m, n, dtype, after, before, want=("before_gamma",))


def test_norms_without_rows(gpu):
    """No rows: nothing is written but the parameters' gradients, which are 0."""
    from tcbnn_amd import head
    s, g = ho.Matrix(None, "f32", 0, 1, 8), ho.empty(8)
    layer = head.BlockNormLayerParam("norms", 0, 8, "f32", "rms", "rms").initialize(s.view, s.view, new_stream_gpu=s.view, output_gpu=s.view)
    layer.initialize_backward(s.view, s.view, s.view, grad_before_gamma_gpu=g)
    layer.forward()
    layer.backward()
    ho.sync()
    assert np.isnan(s.get()).all()
    np.testing.assert_array_equal(g.to_numpy(np.float32, (8,)), np.zeros(8, np.float32))


# --------------------------------------------------------------------------- gated product
# (rows, inputs, features): one value; one row; the halves' 16 rows of a tile and one to each side; whole and ragged tiles; few rows with long sums
GATED = [(1, 1, 1), (1, 16, 10), (1, 4096, 512), (1, 1025, 33), (2, 8, 3), (3, 17, 5), (5, 1032, 264), (7, 33, 1000), (8, 512, 64), (15, 31, 65),
         (16, 64, 16), (17, 72, 15), (31, 2048, 96), (32, 256, 17), (33, 100, 127), (64, 4096, 48), (65, 65, 65), (77, 1023, 129), (128, 128, 128),
         (129, 136, 257), (300, 64, 8), (255, 1000, 511), (513, 96, 300), (4, 1023, 4099), (1000, 1001, 999), (36, 860, 489), (200, 304, 16)]
ACTS = ["none", "relu", "gelu", "silu"]


def _gated(gpu, m, k, n, dtype, activation, bias=True, preact=True, gap=0, stream=None, shift=1):
    from tcbnn_amd import head
    r = rng(m, k, n, len(dtype), len(activation), 2)
    x = ho.Matrix(r.standard_normal((m, k)), dtype, gap, shift=shift)
    w = ho.Matrix(r.standard_normal((2 * n, k)) / np.sqrt(k), dtype, gap, shift=shift)
    b = r.standard_normal(2 * n).astype(np.float32) if bias else None
    y = ho.Matrix(None, dtype, gap, m, n)
    z = ho.Matrix(None, dtype, gap, m, 2 * n) if preact else None
    layer = head.GatedLayerParam("gated", m, k, n, dtype, activation)
    layer.initialize(w.view, b, x.view, output_gpu=y.view, preact_gpu=z.view if preact else None)
    layer.forward(stream)
    ho.sync()
    zw = x.values @ w.values.T + (b.astype(np.float64) if bias else 0.0)
    zerr = (k + 1) * ho.U32 * (np.abs(x.values) @ np.abs(w.values).T + (np.abs(b) if bias else 0.0))
    if preact:
        ho.check(z.get(), zw, zerr + ho.U[dtype] * (np.abs(zw) + zerr) + ho.TINY[dtype], "preact")
    g, u, gerr, uerr = zw[:, :n], zw[:, n:], zerr[:, :n], zerr[:, n:]
    # slopes are below 1.13; the activation itself is good to a few units in the last place of its argument
    a = ho.act(activation, g)
    aerr = 1.13 * gerr + 8 * ho.U32 * np.abs(g)
    ho.check(y.get(), a * u, bo.out_error(a * u, aerr * np.abs(u) + np.abs(a) * uerr + aerr * uerr + ho.U32 * np.abs(a * u), dtype), "output")
    layer.release()


@pytest.mark.parametrize("dtype", ho.DTYPES)
@pytest.mark.parametrize("m,k,n", GATED)
def test_gated(gpu, m, k, n, dtype):
    _gated(gpu, m, k, n, dtype, ACTS[(m + k + n) % 4])


@pytest.mark.parametrize("activation", ACTS)
@pytest.mark.parametrize("m,k,n", [(2, 40, 24), (33, 129, 65), (200, 264, 136)])
def test_gated_epilogues(gpu, m, k, n, activation):
    for dtype in ho.DTYPES:
        for bias, preact in [(False, False), (True, False), (False, True)]:
            _gated(gpu, m, k, n, dtype, activation, bias, preact)


@pytest.mark.parametrize("dtype", ho.DTYPES)
@pytest.mark.parametrize("m,k,n", [(1, 64, 40), (19, 128, 72), (130, 264, 136), (300, 61, 77)])
def test_gated_strides(gpu, m, k, n, dtype):
    _gated(gpu, m, k, n, dtype, "gelu", gap=GAPS[dtype])
    _gated(gpu, m, k, n, dtype, "silu", gap=8, shift=0)


def _gated_kernel(m, k, n, dtype):
    import ctypes as C
    from tcbnn_amd import _lib
    d = _lib.GatedDesc(input=1 << 20, weight=1 << 20, output=1 << 20, rows=m, in_features=k, features=n, dtype=_lib.DTYPES[dtype])
    buf = C.create_string_buffer(160)
    _lib.check(_lib.lib.tcbnn_gated_kernel_name(C.byref(d), buf, 160))
    return buf.value.decode()


# rows at whole 16 bytes: every tile, whole and ragged, with whole steps of the sum and ragged ones; the bf16 plan of each
GATED_WHOLE = [((1, 64, 64), "few_rows_kernel<__bf16, 8>"), ((16, 1048, 72), "few_rows_kernel<__bf16, 8>"), ((3, 264, 8204), "few_rows_kernel<__bf16, 2>"),
               ((17, 1048, 36), "32, 32"), ((33, 8, 4), "32, 32"), ((100, 520, 152), "32, 32"), ((64, 2048, 1024), "32, 32"), ((1024, 512, 512), "64, 64"),
               ((1000, 72, 1500), "64, 64"), ((2040, 136, 1020), "128, 128, 2, 2, 2, 4"), ((2048, 512, 1024), "128, 128, 2, 2, 2, 4"),
               ((2040, 72, 1028), "128, 128, 2, 2, 1, 2"), ((2040, 72, 2052), "128, 128, 2, 2, 1, 1"), ((4096, 64, 2048), "128, 128, 2, 2, 1, 1"),
               ((4000, 200, 2044), "128, 128, 2, 2, 1, 1"), ((4096, 392, 2048), "256, 256"), ((4000, 400, 2044), "256, 256")]


@pytest.mark.parametrize("shape,kernel", GATED_WHOLE)
def test_gated_of_whole_pieces(gpu, shape, kernel):
    assert kernel in _gated_kernel(*shape, "bf16")
    for dtype, activation in (("bf16", "gelu"), ("f16", "none"), ("f32", "silu")):
        _gated(gpu, *shape, dtype, activation, preact=False, shift=0)
    _gated(gpu, *shape, "bf16", "silu", gap=8, shift=0)


@pytest.mark.parametrize("dtype", ho.DTYPES)
@pytest.mark.parametrize("m,k,n", [(3, 4096, 24), (140, 96, 136)])
def test_gated_rows_do_not_mix(gpu, m, k, n, dtype):
    """A NaN row of the input, an infinite row of the gate's weights and one of the rest: one row and two columns of the output."""
    from tcbnn_amd import head
    r = rng(m, k, n)
    xv, wv = r.standard_normal((m, k)), r.standard_normal((2 * n, k))
    xv[1, k - 1] = np.nan
    wv[2, 0] = wv[n + 17, 5] = np.inf
    x, w, y = ho.Matrix(xv, dtype), ho.Matrix(wv, dtype), ho.Matrix(None, dtype, 0, m, n)
    head.GatedLayerParam("gated", m, k, n, dtype, "none").initialize(w.view, None, x.view, output_gpu=y.view).forward()
    ho.sync()
    want = np.ones((m, n), bool)
    want[1] = False
    want[:, [2, 17]] = False
    np.testing.assert_array_equal(np.isfinite(y.get()), want)


def _gated_grad(gpu, m, k, n, dtype, activation, gap=0, want=("x", "w", "b"), shift=1, stream=None):
    from tcbnn_amd import head
    r = rng(m, k, n, len(dtype), len(activation), 3)
    x = ho.Matrix(r.standard_normal((m, k)), dtype, gap, shift=shift)
    w = ho.Matrix(r.standard_normal((2 * n, k)) / np.sqrt(k), dtype, gap, shift=shift)
    z = ho.Matrix(r.standard_normal((m, 2 * n)) * 2, dtype, gap)
    dh = ho.Matrix(r.standard_normal((m, n)), dtype, gap, shift=shift)
    dx, dw, db = ho.Matrix(None, dtype, gap, m, k), ho.Matrix(None, dtype, gap, 2 * n, k), ho.empty(2 * n)
    layer = head.GatedLayerParam("gated", m, k, n, dtype, activation)
    layer.initialize(w.view, None, x.view, preact_gpu=z.view)
    layer.initialize_backward(dh.view, dx.view if "x" in want else None, dw.view if "w" in want else None, db if "b" in want else None)
    layer.backward(stream)
    ho.sync()
    g, u = z.values[:, :n], z.values[:, n:]
    slope, a = ho.slope(activation, g), ho.act(activation, g)
    d = np.concatenate([dh.values * u * slope, dh.values * a], 1)
    # the slope is good to a few units of 1, the activation to as many of its argument
    derr = np.concatenate([np.abs(dh.values * u) * (8 + 2 * np.abs(slope)), np.abs(dh.values) * (8 * np.abs(g) + np.abs(a))], 1) * ho.U32
    used = derr + ho.U[dtype] * (np.abs(d) + derr) + ho.TINY[dtype]  # as the products read it
    if "x" in want:
        exact, terms = d @ w.values, np.abs(d) @ np.abs(w.values)
        err = used @ np.abs(w.values) + 2 * n * ho.U32 * 1.01 * terms
        ho.check(dx.get(), exact, err + ho.U[dtype] * (np.abs(exact) + err) + ho.TINY[dtype], "grad_input")
    if "w" in want:
        exact, terms = d.T @ x.values, np.abs(d).T @ np.abs(x.values)
        err = used.T @ np.abs(x.values) + m * ho.U32 * 1.01 * terms
        ho.check(dw.get(), exact, err + ho.U[dtype] * (np.abs(exact) + err) + ho.TINY[dtype], "grad_weight")
    if "b" in want:
        ho.check(db.to_numpy(np.float32, (2 * n,)), d.sum(0), derr.sum(0) + m * ho.U32 * 1.01 * np.abs(d).sum(0), "grad_bias")
    layer.release()


@pytest.mark.parametrize("dtype", ho.DTYPES)
@pytest.mark.parametrize("m,k,n", GATED)
def test_gated_grad(gpu, m, k, n, dtype):
    _gated_grad(gpu, m, k, n, dtype, ACTS[(m + k + n) % 4])


@pytest.mark.parametrize("dtype", ho.DTYPES)
@pytest.mark.parametrize("m,k,n", [(1, 64, 40), (19, 130, 72), (130, 264, 136), (700, 61, 77), (2100, 40, 600)])
def test_gated_grad_strides_and_single_outputs(gpu, m, k, n, dtype):
    _gated_grad(gpu, m, k, n, dtype, "gelu", gap=GAPS[dtype])
    _gated_grad(gpu, m, k, n, dtype, "none", gap=8, shift=0)
    for want in (("x",), ("w",), ("b",), ("w", "b")):
        _gated_grad(gpu, m, k, n, dtype, "silu", want=want)


# weights' gradients of short sums and many tiles, odd columns among them
@pytest.mark.parametrize("m,k,n", [(16, 2048, 2000), (70, 1024, 3200), (33, 1024, 3203), (500, 520, 5000)])
def test_gated_grad_of_short_sums(gpu, m, k, n):
    for dtype in ho.DTYPES:
        _gated_grad(gpu, m, k, n, dtype, "silu", shift=0)


# large enough that copies of operands that lie anywhere are taken: odd inputs, rows out of wider arrays, odd features, each operand alone
@pytest.mark.parametrize("m,k,n,gap,shift", [(4096, 1023, 1024, 0, 0), (4096, 1024, 1024, 3, 0), (4096, 1024, 1024, 8, 1), (4000, 1025, 1001, 0, 1),
                                             (4096, 2047, 1500, 0, 0), (4096, 2047, 2048, 0, 0)])
def test_gated_on_copies(gpu, m, k, n, gap, shift):
    from tcbnn_amd import _lib
    lib = _lib.lib
    for dtype in ("bf16", "f16"):
        dt = _lib.DTYPES[dtype]
        assert lib.tcbnn_gated_grad_workspace_bytes(m, k, n, dt, 1) > lib.tcbnn_gated_grad_workspace_bytes(m, k, n, dt, 0)
        assert n < 1500 or lib.tcbnn_gated_workspace_bytes(m, k, n, dt) > 0
        assert n < 2048 or lib.tcbnn_gated_workspace_bytes(m, k, n, dt) >= 2 * (k + 1) * (m + 2 * n)  # (both operands')
        _gated(gpu, m, k, n, dtype, "silu", gap=gap, shift=shift)
        _gated_grad(gpu, m, k, n, dtype, "gelu", gap=gap, shift=shift)
    if not gap:
        _gated_grad(gpu, m, k, n, "f32", "silu", shift=shift)


def test_gated_without_rows(gpu):
    from tcbnn_amd import head
    x, dw, db = ho.Matrix(None, "bf16", 0, 32, 8), ho.Matrix(None, "bf16", 0, 32, 8), ho.empty(32)
    layer = head.GatedLayerParam("gated", 0, 8, 16, "bf16").initialize(x.view, None, x.view, output_gpu=x.view, preact_gpu=x.view)
    layer.initialize_backward(x.view, x.view, dw.view, db)
    layer.forward()
    layer.backward()
    ho.sync()
    assert np.isnan(x.get()).all()
    assert (dw.get() == 0).all() and (db.to_numpy(np.float32, (32,)) == 0).all()


# --------------------------------------------------------------------------- linear loss
# (rows, inputs, classes): one value; one row; a part of 16, a tile and one to each side; few rows and long sums; classes in several pieces are below
LOSS = [(1, 1, 1), (1, 16, 10), (1, 4096, 512), (1, 1025, 3), (2, 8, 17), (3, 17, 5), (5, 1032, 1264), (7, 33, 1000), (16, 64, 16), (17, 72, 2), (31, 2048, 96),
        (32, 256, 129), (33, 100, 127), (64, 4096, 48), (65, 65, 65), (77, 1023, 129), (128, 128, 128), (129, 136, 257), (256, 512, 1000), (300, 64, 7),
        (255, 1000, 511), (513, 96, 300), (4, 1023, 4099), (1000, 1001, 999), (3, 5, 4000), (40, 7, 30), (9, 512, 16392), (2100, 64, 40)]


def _loss(gpu, m, k, n, dtype, bias=True, gap=0, shift=1, stream=None, want=("input", "weight", "bias"), scale=1.0, forbidden=(), t=None, mask=-np.inf):
    from tcbnn_amd import head
    r = rng(m, k, n, len(dtype), 4)
    wv = 2.5 * r.standard_normal((n, k)) / np.sqrt(k)
    if t is None:
        t = r.integers(0, n, m).astype(np.int32)
        t[r.random(m) < 0.1] = -1
    xv = r.standard_normal((m, k)) + np.where(r.random(m) < 0.5, 1.0, 0.0)[:, None] * wv[np.clip(t, 0, n - 1)]
    x, w = ho.Matrix(xv, dtype, gap, shift=shift), ho.Matrix(wv, dtype, gap, shift=shift)
    b = r.standard_normal(n).astype(np.float32) if bias else None
    if len(forbidden):
        b[forbidden] = mask
    g = (scale * (0.5 + r.random(m))).astype(np.float32)
    dx, dw, db = ho.Matrix(None, dtype, gap, m, k), ho.Matrix(None, dtype, gap, n, k), ho.empty(n)
    layer = head.LinearLossLayerParam("loss", m, k, n, dtype)
    layer.initialize(w.view, b, x.view, ho.vector(t, np.int32))
    layer.forward(stream)
    ho.sync()
    b64 = b.astype(np.float64) if bias else None
    loss, loss_err, lse, lse_err, z, zerr, p = bo.loss(x.values, w.values, b64, t, g)
    got = layer.download_output()
    ho.check(got["logsumexp"], lse, lse_err, "logsumexp")
    ho.check(got["loss"], loss, loss_err, "loss")
    if want:
        layer.initialize_backward(ho.vector(g), dx.view if "input" in want else None, dw.view if "weight" in want else None, db if "bias" in want else None)
        layer.backward(stream)
        ho.sync()
        exact = bo.loss_grads(x.values, w.values, t, g.astype(np.float64), z, zerr, p, lse, lse_err, dtype)
        for name, buf in (("input", dx), ("weight", dw)):
            if name in want:
                e, err = exact[name]
                ho.check(buf.get(), e, bo.out_error(e, err, dtype), "grad of " + name)
        if "bias" in want:
            e, err = exact["bias"]
            ho.check(db.to_numpy(np.float32, (n,)), e, 1.1 * err + ho.TINY["f32"], "grad of bias")
    layer.release()


@pytest.mark.parametrize("dtype", ho.DTYPES)
@pytest.mark.parametrize("m,k,n", LOSS)
def test_loss(gpu, m, k, n, dtype):
    _loss(gpu, m, k, n, dtype, bias=(m + k + n) % 3 > 0)


@pytest.mark.parametrize("dtype", ho.DTYPES)
@pytest.mark.parametrize("m,k,n", [(1, 64, 40), (19, 128, 72), (130, 264, 136), (300, 61, 77), (40, 24, 1003)])
def test_loss_strides_and_single_outputs(gpu, m, k, n, dtype):
    _loss(gpu, m, k, n, dtype, gap=GAPS[dtype])
    _loss(gpu, m, k, n, dtype, gap=8, shift=0)
    for want in (("input",), ("weight",), ("bias",), ("weight", "bias"), ()):
        _loss(gpu, m, k, n, dtype, want=want, shift=0)


# rows at whole 16 bytes: every tile, whole and ragged
@pytest.mark.parametrize("m,k,n", [(17, 1048, 36), (33, 8, 8), (100, 520, 304), (64, 2048, 2048), (1024, 512, 1024), (1000, 72, 1500), (2040, 136, 1020),
                                   (2048, 512, 1024), (2040, 72, 2052), (2048, 64, 2048), (2000, 200, 2044)])
def test_loss_of_whole_pieces(gpu, m, k, n):
    for dtype in ho.DTYPES:
        _loss(gpu, m, k, n, dtype, shift=0)


@pytest.mark.parametrize("dtype", ho.DTYPES)
def test_loss_in_pieces(gpu, dtype, monkeypatch):
    """Classes whose gradients the workspace does not hold at a time, the last piece a short one."""
    from tcbnn_amd import _lib
    m, k, n = 40000, 24, 1700 if dtype == "f32" else 3400
    assert _lib.lib.tcbnn_linear_loss_grad_workspace_bytes(m, k, n, _lib.DTYPES[dtype], 0) < 1.4 * 2 ** 28
    from tcbnn_amd import head
    r = rng(n)
    x, w = ho.Matrix(r.standard_normal((m, k)), dtype, shift=0), ho.Matrix(r.standard_normal((n, k)) / 4, dtype, shift=0)
    t = r.integers(-1, n, m).astype(np.int32)
    g = (0.5 + r.random(m)).astype(np.float32)
    dx, dw, db = ho.Matrix(None, dtype, 0, m, k), ho.Matrix(None, dtype, 0, n, k), ho.empty(n)
    layer = head.LinearLossLayerParam("loss", m, k, n, dtype).initialize(w.view, None, x.view, ho.vector(t, np.int32))
    layer.initialize_backward(ho.vector(g), dx.view, dw.view, db)
    layer.forward()
    layer.backward()
    ho.sync()
    got, dxv, dwv, dbv = layer.download_output(), dx.get(), dw.get(), db.to_numpy(np.float32, (n,))
    dw_exact = dw_err = db_exact = db_err = 0.0
    for i in range(0, m, 4000):
        rows = slice(i, i + 4000)
        loss, loss_err, lse, lse_err, z, zerr, p = bo.loss(x.values[rows], w.values, None, t[rows], g[rows])
        ho.check(got["loss"][rows], loss, loss_err, "loss")
        e = bo.loss_grads(x.values[rows], w.values, t[rows], g[rows].astype(np.float64), z, zerr, p, lse, lse_err, dtype)
        ho.check(dxv[rows], e["input"][0], bo.out_error(*e["input"], dtype), "grad of input")
        dw_exact, dw_err = dw_exact + e["weight"][0], dw_err + 10 * e["weight"][1]  # (a sum ten times as long)
        db_exact, db_err = db_exact + e["bias"][0], db_err + 10 * e["bias"][1]
    ho.check(dwv, dw_exact, bo.out_error(dw_exact, dw_err, dtype), "grad of weight")
    ho.check(dbv, db_exact, 1.1 * db_err, "grad of bias")
    layer.release()


@pytest.mark.parametrize("m,k,n,gap,shift", [(2048, 1023, 4100, 0, 0), (2048, 1024, 4100, 3, 0), (2047, 1024, 4099, 8, 1), (250, 2047, 8001, 0, 1)])
def test_loss_on_copies(gpu, m, k, n, gap, shift):
    from tcbnn_amd import _lib
    lib = _lib.lib
    for dtype in ("bf16", "f16"):
        assert lib.tcbnn_linear_loss_grad_workspace_bytes(m, k, n, _lib.DTYPES[dtype], 1) > lib.tcbnn_linear_loss_grad_workspace_bytes(m, k, n, _lib.DTYPES[dtype], 0)
        _loss(gpu, m, k, n, dtype, gap=gap, shift=shift)


def test_loss_on_copies_of_pieces(gpu):
    """Weights whose copy is made a piece at a time, forward and backward: against the same values at whole 16 bytes."""
    from tcbnn_amd import head
    m, k, n, dtype = 600, 2047, 70001, "bf16"
    r = rng(k, n)
    xv = r.standard_normal((m, k)).astype(np.float32)
    wv = (r.standard_normal((n, k)) / 20).astype(np.float32)
    t, g = ho.vector(r.integers(-1, n, m), np.int32), ho.vector(np.ones(m))
    out = []
    for pad in (0, 1):  # (a column of zeros more is at whole 16 bytes)
        x, w = (ho.Matrix(np.pad(v, ((0, 0), (0, pad))), dtype, shift=0) for v in (xv, wv))
        dx, dw = ho.Matrix(None, dtype, 0, m, k + pad, shift=0), ho.Matrix(None, dtype, 0, n, k + pad, shift=0)
        layer = head.LinearLossLayerParam("loss", m, k + pad, n, dtype).initialize(w.view, None, x.view, t)
        layer.initialize_backward(g, dx.view, dw.view)
        layer.forward()
        layer.backward()
        ho.sync()
        got = layer.download_output()
        out.append((got["loss"], got["logsumexp"], dx.get()[:, :k], dw.get()[:, :k]))
        layer.release()
    for a, b in zip(*out):
        np.testing.assert_array_equal(a, b)


def test_loss_of_forbidden_classes(gpu):
    """A bias of -inf: no share in the sums, no gradient; a row whose class is forbidden."""
    for dtype in ho.DTYPES:
        for m, k, n in ((1, 64, 100), (12, 40, 700), (150, 72, 1000)):
            r = rng(m, n)
            t = r.integers(n // 2, n, m).astype(np.int32)
            t[::5] = -1
            _loss(gpu, m, k, n, dtype, forbidden=np.arange(n // 2), t=t)


# input gradients of few rows and long sums, in many parts
@pytest.mark.parametrize("m,k,n", [(5, 560, 20889), (21, 80, 17700), (60, 304, 30000), (64, 1024, 4000), (65, 160, 22985), (100, 2488, 9000), (128, 520, 20003)])
def test_loss_of_few_rows_and_many_classes(gpu, m, k, n):
    for dtype in ho.DTYPES:
        _loss(gpu, m, k, n, dtype, shift=0)
    _loss(gpu, m, k, n, "bf16", gap=8, shift=0, want=("input",))


# short sums and many tiles, of the logits and of the weights' gradients; the largest tiles
@pytest.mark.parametrize("m,k,n", [(16, 2048, 4000), (40, 1024, 8000), (40, 1024, 8003), (300, 520, 12500), (2048, 64, 4096), (2040, 72, 4100), (1100, 504, 6000), (4096, 1040, 2048)])
def test_loss_of_short_sums(gpu, m, k, n):
    for dtype in ho.DTYPES:
        _loss(gpu, m, k, n, dtype, shift=0)


@pytest.mark.parametrize("dtype", ho.DTYPES)
@pytest.mark.parametrize("m,k,n,shift", [(1, 64, 100, 1), (3, 40, 70, 0), (12, 40, 700, 1), (40, 24, 130, 0), (150, 72, 1000, 1), (1024, 64, 1024, 0), (2048, 64, 2048, 0)])
def test_loss_of_classes_masked_by_the_lowest_value(gpu, m, k, n, shift, dtype):
    """A bias of the lowest finite value, over whole tiles: as good as -inf."""
    _loss(gpu, m, k, n, dtype, shift=shift, forbidden=np.arange(n - n // 2, n), t=rng(m, n).integers(-1, n - n // 2, m).astype(np.int32), mask=np.finfo(np.float32).min)


@pytest.mark.parametrize("m,k,n", [(2, 24, 40), (9, 24, 40), (40, 24, 300), (2048, 64, 2048)])
def test_loss_of_rows_far_from_0(gpu, m, k, n):
    """Every class at the lowest finite value, or at the highest: log(classes), and gradients that are numbers."""
    from tcbnn_amd import head
    for dtype in ho.DTYPES:
        for value in (np.finfo(np.float32).min, 3e38):
            r = rng(m, n)
            x, w = (ho.Matrix(r.standard_normal((rows, k)), dtype, shift=0) for rows in (m, n))
            dx, dw, db = ho.Matrix(None, dtype, 0, m, k, shift=0), ho.Matrix(None, dtype, 0, n, k, shift=0), ho.empty(n)
            layer = head.LinearLossLayerParam("loss", m, k, n, dtype)
            layer.initialize(w.view, np.full(n, value, np.float32), x.view, ho.vector(r.integers(0, n, m), np.int32))
            layer.initialize_backward(ho.vector(np.full(m, 1.0 / n)), dx.view, dw.view, db)
            layer.forward()
            layer.backward()
            ho.sync()
            out = layer.download_output()
            assert (out["logsumexp"] == np.float32(value)).all()
            # (the sum is of n ones, its logarithm off by a few units)
            np.testing.assert_allclose(out["loss"], np.log(n), rtol=2.0 ** -20)
            assert np.isfinite(dx.get()).all() and np.isfinite(dw.get()).all() and np.isfinite(db.to_numpy(np.float32, (n,))).all()
            layer.release()


@pytest.mark.parametrize("m,k,n", [(1, 24, 14), (4, 64, 300), (12, 64, 40), (70, 64, 500), (2048, 64, 4096)])
def test_loss_gradient_of_a_nearly_certain_class(gpu, m, k, n):
    """p - 1 of a given class whose p is about 1 - e^-7: with the loss it carries that one's error, without it logsumexp's."""
    import ctypes as C
    from tcbnn_amd import _lib, head
    r = rng(m, k, n)
    t = np.full(m, n // 3, np.int32)
    # two inputs of whole sixteenths: logits are exact in fp32
    wv, xv = np.zeros((n, k)), np.zeros((m, k))
    wv[:, 0], xv[:, 0] = r.integers(0, 16, n) / 16.0, 1.0
    wv[t, 1], xv[:, 1] = 1.0, np.round(16 * (8 + np.log(n))) / 16
    x, w = ho.Matrix(xv, "f32", shift=0), ho.Matrix(wv, "f32", shift=0)
    z = x.values @ w.values.T
    given = np.arange(n)[None, :] == t[:, None]
    e = np.exp(z - z.max(1, keepdims=True))
    d = e / e.sum(1, keepdims=True)
    d[given] = -np.where(given, 0.0, e).sum(1) / e.sum(1)
    lse = np.log(e.sum(1, keepdims=True)) + z.max(1, keepdims=True)
    layer = head.LinearLossLayerParam("loss", m, k, n, "f32").initialize(w.view, None, x.view, ho.vector(t, np.int32))
    for with_loss in (True, False):
        db = ho.empty(n)
        layer.initialize_backward(ho.vector(np.ones(m)), None, None, db)
        layer.forward()
        desc = layer._grad_desc
        desc.loss = desc.loss if with_loss else None
        _lib.check(_lib.lib.tcbnn_linear_loss_backward(C.byref(desc), None))
        ho.sync()
        # of the other classes: logsumexp's rounding and one like it, exp's argument and some units; of the given one: the loss is the logarithm of a
        # sum a little above 1, to which at most 128 roundings of its size go on the way
        units = np.where(given, 128 + (0 if with_loss else 4 * lse + 16), np.abs(d) * (160 + 4 * lse + 4 * np.abs(z - lse)))
        ho.check(db.to_numpy(np.float32, (n,)), d.sum(0), ho.U32 * (units.sum(0) + (m + 4) * np.abs(d).sum(0)), "with the loss" if with_loss else "without")
    layer.release()


def test_loss_of_degenerate_rows(gpu):
    """Every class forbidden; a forbidden class given; a class that there is not; a NaN and an infinite logit; rows without a class."""
    from tcbnn_amd import head
    for dtype in ho.DTYPES:
        for m, k, n in ((8, 24, 40), (40, 24, 300)):
            for all_forbidden in (False, True):
                r = rng(m, n)
                xv, wv = r.standard_normal((m, k)), r.standard_normal((n, k))
                xv[0, 3], xv[1, 3] = np.nan, np.inf
                wv[:, 3] = np.abs(wv[:, 3]) + 0.1
                b = np.zeros(n, np.float32)
                b[:3] = -np.inf
                if all_forbidden:
                    b[:] = -np.inf
                    xv[:2] = 1.0
                t = r.integers(3, n, m).astype(np.int32)
                t[2], t[3], t[4], t[5] = 1, n, -1, -7
                x, w = ho.Matrix(xv, dtype), ho.Matrix(wv, dtype)
                dx = ho.Matrix(None, dtype, 0, m, k)
                layer = head.LinearLossLayerParam("loss", m, k, n, dtype).initialize(w.view, b, x.view, ho.vector(t, np.int32))
                layer.initialize_backward(ho.vector(np.ones(m)), dx.view)
                layer.forward()
                layer.backward()
                ho.sync()
                out, d = layer.download_output(), dx.get()
                if all_forbidden:
                    assert (out["logsumexp"] == -np.inf).all()
                    want = np.full(m, np.inf)
                    want[3], want[4:6] = np.nan, 0
                    np.testing.assert_array_equal(out["loss"], want)
                    d = np.delete(d, 3, 0)  # (a class that there is not is told by its loss)
                    assert (d == 0).all()
                    continue
                assert np.isnan(out["loss"][:2]).all() and np.isnan(out["logsumexp"][:2]).all() and np.isnan(d[:2]).all()
                assert out["loss"][2] == np.inf and np.isnan(out["loss"][3]) and np.isfinite(out["logsumexp"][2:]).all()
                assert np.isnan(d[3]).all() and (out["loss"][4:6] == 0).all() and (d[4:6] == 0).all()
                assert np.isfinite(out["loss"][6:]).all() and np.isfinite(d[6:]).all() and np.isfinite(d[2]).all()


@pytest.mark.parametrize("scale", [2.0 ** -40, 2.0 ** -20, 1.0 / 8192, 100.0])
def test_loss_gradients_of_any_size(gpu, scale):
    """f16: what d is scaled by does not show, but in what leaves as f16."""
    for dtype in ("f16", "bf16"):
        _loss(gpu, 70, 64, 500, dtype, scale=scale)


def test_loss_without_rows(gpu):
    from tcbnn_amd import head
    x, dw, db = ho.Matrix(None, "bf16", 0, 32, 8), ho.Matrix(None, "bf16", 0, 32, 8), ho.empty(32)
    layer = head.LinearLossLayerParam("loss", 0, 8, 32, "bf16").initialize(x.view, None, x.view, ho.empty(1))
    layer.initialize_backward(db, x.view, dw.view, db)
    layer.forward()
    layer.backward()
    ho.sync()
    assert np.isnan(x.get()).all()
    assert (dw.get() == 0).all() and (db.to_numpy(np.float32, (32,)) == 0).all()
