"""The float head on the GPU against definitions in 64 bits: linear layers, layer norms, log probabilities, and the
gradient of each; sizes around those where the kernels change, odd sizes, strides, empty and degenerate inputs."""
import numpy as np
import pytest

from tests import headops as ho

pytestmark = pytest.mark.gpu

GAPS = {"f32": 1, "bf16": 3, "f16": 5}


def rng(*seed):
    return np.random.default_rng([abs(int(s)) for s in seed])


# --------------------------------------------------------------------------- linear
# (rows, inputs, outputs): one value; one row; the widths of matrix instructions and one to each side; whole and ragged
# tiles; few rows with long sums; more rows than a tile
LINEAR = [(1, 1, 1), (1, 16, 10), (1, 4096, 512), (1, 1025, 33), (2, 8, 3), (3, 17, 5), (5, 1032, 264), (7, 33, 1000),
          (8, 512, 64), (15, 31, 65), (16, 64, 16), (17, 72, 130), (31, 2048, 96), (32, 256, 129), (33, 100, 127),
          (64, 4096, 48), (65, 65, 65), (77, 1023, 129), (127, 200, 128), (128, 128, 128), (129, 136, 257),
          (256, 512, 1000), (300, 64, 8), (255, 1000, 511), (513, 96, 300), (1000, 24, 1030), (4, 1023, 4099), (8, 16385, 33), (1000, 1001, 999),
          (36, 860, 489), (200, 304, 16), (128, 520, 512)]


def _linear(gpu, m, k, n, dtype, activation, bias=True, residual=True, preact=True, gap=0, in_place=False, stream=None, shift=1):
    from tcbnn_amd import head
    r = rng(m, k, n, len(dtype), len(activation))
    x = ho.Matrix(r.standard_normal((m, k)), dtype, gap, shift=shift)
    w = ho.Matrix(r.standard_normal((n, k)) / np.sqrt(k), dtype, gap, shift=shift)
    b = r.standard_normal(n).astype(np.float32) if bias else None
    res = ho.Matrix(r.standard_normal((m, n)), dtype, gap) if residual else None
    rv = res.values if residual else 0.0
    y = res if in_place else ho.Matrix(None, dtype, gap, m, n)
    z = ho.Matrix(None, dtype, gap, m, n) if preact else None
    layer = head.LinearLayerParam("linear", m, k, n, dtype, activation)
    layer.initialize(w.view, b, x.view, residual_gpu=res.view if residual else None, output_gpu=y.view,
                     preact_gpu=z.view if preact else None)
    layer.forward(stream)
    ho.sync()
    zw = x.values @ w.values.T + (b.astype(np.float64) if bias else 0.0)
    zerr = (k + 1) * ho.U32 * (np.abs(x.values) @ np.abs(w.values).T + (np.abs(b) if bias else 0.0))
    if preact:
        ho.check(z.get(), zw, zerr + ho.U[dtype] * (np.abs(zw) + zerr) + ho.TINY[dtype], "preact")
    yw = ho.act(activation, zw) + rv
    # slopes are below 1.13; the activation itself is good to a few units in the last place of its argument
    yerr = 1.13 * zerr + 8 * ho.U32 * (np.abs(zw) + np.abs(rv))
    ho.check(y.get(), yw, yerr + ho.U[dtype] * (np.abs(yw) + yerr) + ho.TINY[dtype], "output")
    layer.release()


@pytest.mark.parametrize("dtype", ho.DTYPES)
@pytest.mark.parametrize("m,k,n", LINEAR)
def test_linear(gpu, m, k, n, dtype):
    _linear(gpu, m, k, n, dtype, ["none", "relu", "gelu", "silu"][(m + k + n) % 4])


@pytest.mark.parametrize("activation", ["none", "relu", "gelu", "silu"])
@pytest.mark.parametrize("m,k,n", [(2, 40, 24), (33, 129, 65), (200, 264, 136)])
def test_linear_epilogues(gpu, m, k, n, activation):
    for dtype in ho.DTYPES:
        for bias, residual, preact in [(False, False, False), (True, False, True), (False, True, False)]:
            _linear(gpu, m, k, n, dtype, activation, bias, residual, preact)


@pytest.mark.parametrize("dtype", ho.DTYPES)
@pytest.mark.parametrize("m,k,n", [(1, 64, 40), (19, 128, 72), (130, 264, 136), (300, 61, 77)])
def test_linear_strides_and_output_over_residual(gpu, m, k, n, dtype):
    _linear(gpu, m, k, n, dtype, "gelu", gap=GAPS[dtype])
    _linear(gpu, m, k, n, dtype, "silu", gap=8, in_place=True)


@pytest.mark.parametrize("dtype", ho.DTYPES)
@pytest.mark.parametrize("m,k,n", [(3, 4096, 24), (140, 96, 136)])
def test_linear_rows_do_not_mix(gpu, m, k, n, dtype):
    """A NaN row of the input, an infinite row of the weight: one row and one column of the output, nothing else."""
    from tcbnn_amd import head
    r = rng(m, k, n)
    xv, wv = r.standard_normal((m, k)), r.standard_normal((n, k))
    xv[1, k - 1] = np.nan
    wv[2, 0] = np.inf
    x, w, y = ho.Matrix(xv, dtype), ho.Matrix(wv, dtype), ho.Matrix(None, dtype, 0, m, n)
    head.LinearLayerParam("linear", m, k, n, dtype).initialize(w.view, None, x.view, output_gpu=y.view).forward()
    ho.sync()
    finite = np.isfinite(y.get())
    want = np.ones((m, n), bool)
    want[1] = False
    want[:, 2] = False
    np.testing.assert_array_equal(finite, want)


def _linear_grad(gpu, m, k, n, dtype, activation, gap=0, want=("x", "w", "b"), shift=1):
    from tcbnn_amd import head
    r = rng(m, k, n, len(dtype), len(activation), 1)
    x = ho.Matrix(r.standard_normal((m, k)), dtype, gap, shift=shift)
    w = ho.Matrix(r.standard_normal((n, k)) / np.sqrt(k), dtype, gap, shift=shift)
    z = ho.Matrix(r.standard_normal((m, n)) * 2, dtype, gap)
    dy = ho.Matrix(r.standard_normal((m, n)), dtype, gap, shift=shift)
    dx, dw, db = ho.Matrix(None, dtype, gap, m, k), ho.Matrix(None, dtype, gap, n, k), ho.empty(n)
    layer = head.LinearLayerParam("linear", m, k, n, dtype, activation)
    layer.initialize(w.view, None, x.view, preact_gpu=z.view if activation != "none" else None)
    layer.initialize_backward(dy.view, dx.view if "x" in want else None, dw.view if "w" in want else None,
                              db if "b" in want else None)
    layer.backward()
    ho.sync()
    g = dy.values * ho.slope(activation, z.values)
    gerr = 8 * ho.U32 * np.abs(dy.values) * (0 if activation == "none" else 1)  # the slope, good to a few units of 1
    used = gerr + (ho.U[dtype] * (np.abs(g) + gerr) + ho.TINY[dtype] if activation != "none" else 0.0)  # as the products read it
    if "x" in want:
        exact, terms = g @ w.values, np.abs(g) @ np.abs(w.values)
        err = used @ np.abs(w.values) + n * ho.U32 * 1.01 * terms
        ho.check(dx.get(), exact, err + ho.U[dtype] * (np.abs(exact) + err) + ho.TINY[dtype], "grad_input")
    if "w" in want:
        exact, terms = g.T @ x.values, np.abs(g).T @ np.abs(x.values)
        err = used.T @ np.abs(x.values) + m * ho.U32 * 1.01 * terms
        ho.check(dw.get(), exact, err + ho.U[dtype] * (np.abs(exact) + err) + ho.TINY[dtype], "grad_weight")
    if "b" in want:
        ho.check(db.to_numpy(np.float32, (n,)), g.sum(0), gerr.sum(0) + m * ho.U32 * 1.01 * np.abs(g).sum(0), "grad_bias")
    layer.release()


@pytest.mark.parametrize("dtype", ho.DTYPES)
@pytest.mark.parametrize("m,k,n", LINEAR)
def test_linear_grad(gpu, m, k, n, dtype):
    _linear_grad(gpu, m, k, n, dtype, ["none", "relu", "gelu", "silu"][(m + k + n) % 4])


@pytest.mark.parametrize("dtype", ho.DTYPES)
@pytest.mark.parametrize("m,k,n", [(1, 64, 40), (19, 130, 72), (130, 264, 136), (700, 61, 77)])
def test_linear_grad_strides_and_single_outputs(gpu, m, k, n, dtype):
    _linear_grad(gpu, m, k, n, dtype, "gelu", gap=GAPS[dtype])
    _linear_grad(gpu, m, k, n, dtype, "none", gap=8)
    for want in (("x",), ("w",), ("b",), ("w", "b")):
        _linear_grad(gpu, m, k, n, dtype, "silu", want=want)
        _linear_grad(gpu, m, k, n, dtype, "none", want=want)


def _kernel(m, k, n, dtype):
    import ctypes as C
    from tcbnn_amd import _lib
    dt = _lib.DTYPES[dtype]
    d = _lib.LinearDesc(input=1 << 20, weight=1 << 20, output=1 << 20, rows=m, in_features=k, out_features=n, dtype=dt, workspace=1 << 20,
                        workspace_bytes=_lib.lib.tcbnn_linear_workspace_bytes(m, k, n, dt))
    buf = C.create_string_buffer(160)
    _lib.check(_lib.lib.tcbnn_linear_kernel_name(C.byref(d), buf, 160))
    return buf.value.decode()


# rows at whole 16 bytes: every tile, with whole tiles and ragged ones, whole steps of the sum and ragged ones, sums of one step, of fewer
# than the tile keeps under way and of many; the bf16 plan of each
WHOLE = [((1, 64, 64), "few_rows_kernel<__bf16, 8>"), ((16, 1048, 72), "few_rows_kernel<__bf16, 8>"), ((3, 264, 16408), "few_rows_kernel<__bf16, 2>"),
         ((9, 512, 16392), "few_rows_kernel<__bf16, 2>"), ((16, 1032, 8200), "32, 32"), ((5, 16384, 64), "join"), ((17, 1048, 72), "32, 32"), ((33, 8, 8), "32, 32"), ((40, 64, 64), "32, 32"),
         ((100, 520, 304), "32, 32"), ((300, 256, 520), "32, 32"), ((64, 2048, 2048), "32, 32"), ((64, 16384, 64), "join"),
         ((128, 4096, 136), "join"), ((1024, 512, 1024), "64, 64"), ((1000, 72, 3000), "64, 64"), ((1016, 1032, 1048), "64, 64"),
         ((2040, 136, 2040), "128, 128, 2, 2, 2, 4"), ((2048, 512, 2048), "128, 128, 2, 2, 2, 4"), ((2040, 72, 4104), "128, 128, 2, 2, 1, 2"),
         ((3000, 200, 3000), "128, 128, 2, 2, 1, 2"), ((4096, 64, 4096), "256, 256"), ((4000, 200, 4088), "256, 256")]


@pytest.mark.parametrize("shape,kernel", WHOLE)
def test_linear_of_whole_pieces(gpu, shape, kernel):
    assert kernel in _kernel(*shape, "bf16")
    for dtype, activation in (("bf16", "gelu"), ("f16", "none"), ("f32", "silu")):
        _linear(gpu, *shape, dtype, activation, preact=False, shift=0)
    _linear(gpu, *shape, "bf16", "relu", gap=8, in_place=True, shift=0)


# the same tiles for the gradients: (rows, sum, columns) of grad_input, then of grad_weight
WHOLE_GRADS = [((40, 64, 64), "32, 32"), ((100, 304, 520), "32, 32"), ((64, 2048, 2048), "32, 32"), ((64, 16384, 64), "join"), ((1000, 72, 3000), "64, 64"),
               ((1016, 1032, 1048), "64, 64"), ((2040, 136, 2040), "128, 128, 2, 2, 2, 4"), ((2040, 72, 4104), "128, 128, 2, 2, 1, 2"),
               ((4000, 72, 4088), "256, 256")]


@pytest.mark.parametrize("shape,kernel", WHOLE_GRADS)
def test_linear_grad_of_whole_pieces(gpu, shape, kernel):
    assert kernel in _kernel(*shape, "bf16")
    rows, total, cols = shape
    for dtype, activation in (("bf16", "none"), ("f16", "gelu"), ("f32", "relu")):
        _linear_grad(gpu, rows, cols, total, dtype, activation, want=("x",), shift=0)
        _linear_grad(gpu, total, cols, rows, dtype, activation, want=("w",), shift=0)
    _linear_grad(gpu, min(rows, 300), min(cols, 520), min(total, 200), "bf16", "silu", gap=8, shift=0)


def test_linear_sums_in_one_order(gpu):
    """The same bits in every call, whatever was in the workspace."""
    from tcbnn_amd import head
    r = rng(77)
    m, k, n = 64, 16384, 64
    x, w, z, dy = (ho.Matrix(r.standard_normal(s), "bf16", shift=0) for s in ((m, k), (n, k), (m, n), (m, n)))
    y, dx, dw, db = (ho.Matrix(None, "bf16", 0, *s, shift=0) for s in ((m, n), (m, k), (n, k), (1, 2 * n)))
    layer = head.LinearLayerParam("linear", m, k, n, "bf16", "gelu").initialize(w.view, None, x.view, output_gpu=y.view, preact_gpu=z.view)
    layer.initialize_backward(dy.view, dx.view, dw.view, db.view)
    first = None
    for fill in (0, 0xFF, 0x3C):
        for buf in layer._owned:
            buf.fill(fill)
        layer.backward()
        layer.forward()
        ho.sync()
        bits = [a.buf.to_numpy(np.uint16, (a.shape[0] * a.shape[1],)) for a in (y, dx, dw, db)]
        first = first or bits
        for a, b in zip(bits, first):
            np.testing.assert_array_equal(a, b)
        z.buf.upload(head.encode(z.values.astype(np.float32), "bf16"))
    layer.release()


class _Apart:
    """Rows so far apart that their offsets pass 32 bits, on the device."""

    def __init__(self, values, dtype, ld):
        from tcbnn_amd import _lib, head
        self.rows, self.cols, self.ld, self.dtype = *values.shape, ld, dtype
        self.size = 4 if dtype == "f32" else 2
        self.buf = ho.DeviceBuffer(self.size * (ld * (self.rows - 1) + self.cols))
        self.view = ho.DeviceView(self.buf.ptr, self.buf.nbytes, ld, self.buf)
        bits = head.encode(values, dtype)
        self.values = head.decode(bits, dtype).astype(np.float64)
        for i in range(self.rows):
            row = np.ascontiguousarray(bits[i])
            _lib.hip_check(_lib.hip.hipMemcpy(self.buf.ptr + self.size * ld * i, row.ctypes.data, row.nbytes, _lib.H2D))

    def get(self):
        from tcbnn_amd import _lib, head
        out = np.empty((self.rows, self.cols), head.storage(self.dtype))
        for i in range(self.rows):
            row = np.empty(self.cols, out.dtype)
            _lib.hip_check(_lib.hip.hipMemcpy(row.ctypes.data, self.buf.ptr + self.size * self.ld * i, row.nbytes, _lib.D2H))
            out[i] = row
        return head.decode(out, self.dtype).astype(np.float64)


@pytest.mark.parametrize("rows,ld", [(3, (1 << 30) + 8), (40, (1 << 26) + 4)])
def test_offsets_past_32_bits(gpu, rows, ld):
    """Rows 2 GiB (or 128 MiB, in more rows than the kernel for few rows takes) apart: each operator reads and writes them."""
    from tcbnn_amd import head
    r = rng(rows)
    n = 72
    x = _Apart(r.standard_normal((rows, n)).astype(np.float32), "bf16", ld)
    gamma, beta = np.ones(n, np.float32), np.zeros(n, np.float32)
    mean, rstd = ho.empty(rows), ho.empty(rows)
    y = ho.Matrix(None, "bf16", 0, rows, n)
    norm = head.LayerNormLayerParam("norm", rows, n, "bf16", EPS).initialize(gamma, beta, x.view, output_gpu=y.view, mean_gpu=mean, rstd_gpu=rstd)
    norm.forward()
    ho.sync()
    _check_norm(x.values, gamma.astype(np.float64), beta.astype(np.float64), y.get(), mean.to_numpy(np.float32, (rows,)),
                rstd.to_numpy(np.float32, (rows,)), "bf16")
    w = ho.Matrix(r.standard_normal((24, n)), "bf16")
    z = ho.Matrix(None, "bf16", 0, rows, 24)
    head.LinearLayerParam("linear", rows, n, 24, "bf16").initialize(w.view, None, x.view, output_gpu=z.view).forward()
    ho.sync()
    exact, terms = x.values @ w.values.T, np.abs(x.values) @ np.abs(w.values).T
    ho.check(z.get(), exact, n * ho.U32 * terms + ho.U["bf16"] * (np.abs(exact) + terms * n * ho.U32), "linear")
    lin = head.LinearLayerParam("linear", rows, 24, n, "bf16").initialize(ho.Matrix(r.standard_normal((n, 24)), "bf16").view, None, z.view)
    dw = ho.Matrix(None, "bf16", 0, n, 24)
    lin.initialize_backward(x.view, None, dw.view, None)  # (the far rows as grad_output)
    lin.backward()
    ho.sync()
    exact, terms = x.values.T @ z.get(), np.abs(x.values).T @ np.abs(z.get())
    ho.check(dw.get(), exact, rows * ho.U32 * terms + ho.U["bf16"] * (np.abs(exact) + terms * rows * ho.U32), "grad_weight")
    t = r.integers(0, n, rows).astype(np.int32)
    lp = head.LogProbsLayerParam("logprobs", rows, n, 4, "bf16").initialize(x.view, ho.vector(t, np.int32))
    lp.initialize_backward(ho.vector(np.ones(rows)), None, x.view)
    lp.forward()
    ho.sync()
    want = [ho.logprobs(x.values[i], int(t[i]), 4) for i in range(rows)]
    got = lp.download_output()
    np.testing.assert_array_equal(got["top_index"], np.stack([v[4] for v in want]))
    np.testing.assert_allclose(got["logprob"], [v[0] for v in want], atol=1e-5)
    lp.backward()
    ho.sync()
    p = np.exp(x.values - np.array([v[2] for v in want])[:, None])
    hot = (np.arange(n) == t[:, None]) - p
    ho.check(x.get(), hot, 2 * ho.U["bf16"] * np.abs(hot) + 1e-6, "grad_logits")
    for layer in (norm, lin, lp):
        layer.release()
    x.buf.free()


def test_linear_split_sums_of_far_rows(gpu):
    """A long sum, split among workgroups, over weight rows that are read element by element; the gradients of such a layer."""
    from tcbnn_amd import head
    m, k, n = 40, 16390, 24
    r = rng(m, k, n)
    w = _Apart((r.standard_normal((n, k)) / np.sqrt(k)).astype(np.float32), "bf16", (1 << 22) + 8)
    x, dy = ho.Matrix(r.standard_normal((m, k)), "bf16"), ho.Matrix(r.standard_normal((m, n)), "bf16")
    y, dx, dw = ho.Matrix(None, "bf16", 0, m, n), ho.Matrix(None, "bf16", 0, m, k), ho.Matrix(None, "bf16", 0, n, k)
    layer = head.LinearLayerParam("linear", m, k, n, "bf16").initialize(w.view, None, x.view, output_gpu=y.view)
    layer.initialize_backward(dy.view, dx.view, dw.view)
    assert layer._desc.workspace_bytes > 0
    layer.forward()
    layer.backward()
    ho.sync()
    for got, a, b in ((y, x.values, w.values.T), (dx, dy.values, w.values), (dw, dy.values.T, x.values)):
        exact, terms = a @ b, np.abs(a) @ np.abs(b)
        err = (a.shape[1] + 1) * ho.U32 * terms
        ho.check(got.get(), exact, err + ho.U["bf16"] * (np.abs(exact) + err) + ho.TINY["bf16"])
    layer.release()
    w.buf.free()


def test_linear_of_more_rows_than_a_launch_has(gpu):
    """Rows shorter than 16 bytes go through tiles of 32 whatever their number: 2^29 of them are 2^32 threads."""
    from tcbnn_amd import head
    m, k, n = (1 << 29) + 77, 4, 4
    x, y = ho.DeviceBuffer(2 * m * k), ho.DeviceBuffer(2 * m * n)
    x.fill(0x3c)
    y.fill(0x7f)
    value = np.float64(np.uint16(0x3c3c).view(np.float16))
    w = np.arange(1, 17, dtype=np.float32).reshape(n, k) / 16
    layer = head.LinearLayerParam("linear", m, k, n, "f16").initialize(w, None, x, output_gpu=y)
    layer.initialize_backward(x, y)
    for run, sums in ((layer.forward, w.sum(1)), (layer.backward, w.sum(0))):
        y.fill(0x7f)
        run()
        ho.sync()
        for first in (0, 77, m // 2, m - 100):
            got = ho.DeviceView(y.ptr + 2 * n * first, 2 * n * 100).to_numpy(np.float16, (100, n)).astype(np.float64)
            np.testing.assert_allclose(got, np.tile(value * sums, (100, 1)), rtol=2 * ho.U["f16"])
    layer.release()
    x.free()
    y.free()


def test_bias_gradients_of_most_outputs_without_rows(gpu):
    import ctypes as C
    from tcbnn_amd import _lib
    n = 1 << 28
    db = ho.DeviceBuffer(4 * n)
    db.fill(0x7f)
    d = _lib.LinearGradDesc(grad_bias=db.ptr, rows=0, in_features=1, out_features=n, dtype=1)
    _lib.check(_lib.lib.tcbnn_linear_backward(C.byref(d), None))
    ho.sync()
    assert not db.to_numpy(np.uint32, (n,)).any()
    db.free()


def test_linear_without_rows(gpu):
    from tcbnn_amd import head
    x, w = ho.Matrix(None, "bf16", 0, 0, 24), ho.Matrix(np.ones((16, 24)), "bf16")
    y, dw, db = ho.Matrix(None, "bf16", 0, 0, 16), ho.Matrix(None, "bf16", 0, 16, 24), ho.empty(16)
    layer = head.LinearLayerParam("linear", 0, 24, 16, "bf16", "gelu")
    layer.initialize(w.view, None, x.view, output_gpu=y.view, save_preact=True)
    layer.initialize_backward(y.view, x.view, dw.view, db)
    layer.forward()
    layer.backward()
    ho.sync()
    assert not dw.get().any() and not db.to_numpy(np.float32, (16,)).any()


# --------------------------------------------------------------------------- layer norm
NORM = [(1, 1), (3, 2), (5, 7), (70, 64), (4, 100), (300, 128), (2, 512), (9, 513), (33, 1000), (65, 1023), (3, 1024),
        (1, 4096), (17, 4097), (3, 8192), (2, 8195), (5, 16384), (2, 20001), (1, 65536)]
EPS = 1e-5


def _norm_inputs(m, n, dtype, gap, offset=0.5):
    r = rng(m, n, len(dtype))
    x = ho.Matrix(2.0 * r.standard_normal((m, n)) + offset, dtype, gap)
    gamma, beta = (1 + 0.2 * r.standard_normal(n)).astype(np.float32), r.standard_normal(n).astype(np.float32)
    return r, x, gamma, beta


def _check_norm(x, gamma, beta, y, mean, rstd, dtype):
    n = x.shape[1]
    yw, mw, rw = ho.norm(x, gamma, beta, EPS)
    # sums of n terms over at least 64 lanes: n / 64 terms in a row at most, and the steps that join the lanes
    depth = n / 64 + 24
    merr = depth * ho.U32 * np.abs(x).mean(1)
    ho.check(mean, mw, merr, "mean")
    # the variance's own relative error, and what the mean's adds (its square, and nothing in first order)
    verr = (2 * depth + 6) * ho.U32 + (merr * rw) ** 2
    ho.check(rstd, rw, rw * (0.5 * verr + 4 * ho.U32), "rstd")
    xh = (x - mw[:, None]) * rw[:, None]
    err = (np.abs(gamma) * (np.abs(xh) * (0.5 * verr + 8 * ho.U32)[:, None] + ((merr + ho.U32 * np.abs(x).max(1)) * rw)[:, None])
           + 2 * ho.U32 * np.abs(yw))
    ho.check(y, yw, err + ho.U[dtype] * (np.abs(yw) + err) + ho.TINY[dtype], "output")


@pytest.mark.parametrize("dtype", ho.DTYPES)
@pytest.mark.parametrize("m,n", NORM)
def test_layernorm(gpu, m, n, dtype):
    from tcbnn_amd import head
    for gap in (0, GAPS[dtype], 8):
        r, x, gamma, beta = _norm_inputs(m, n, dtype, gap)
        y = ho.Matrix(None, dtype, gap, m, n)
        layer = head.LayerNormLayerParam("norm", m, n, dtype, EPS).initialize(gamma, beta, x.view, output_gpu=y.view)
        layer.forward()
        ho.sync()
        _check_norm(x.values, gamma.astype(np.float64), beta.astype(np.float64), y.get(), layer.mean_gpu.to_numpy(np.float32, (m,)),
                    layer.rstd_gpu.to_numpy(np.float32, (m,)), dtype)
        layer.release()


@pytest.mark.parametrize("n", [64, 1000, 5000])
def test_layernorm_far_from_zero_and_in_place(gpu, n):
    """A variance that is small beside the mean's square, as only sums about the mean hold it; output over input; no
    parameters; a row of equal values."""
    from tcbnn_amd import head
    m = 6
    r = rng(n)
    v = 1000.0 + r.standard_normal((m, n))
    v[2] = 3.0
    x = ho.Matrix(v, "f32")
    layer = head.LayerNormLayerParam("norm", m, n, "f32", EPS).initialize(None, None, x.view, output_gpu=x.view)
    layer.forward()
    ho.sync()
    _check_norm(x.values, np.ones(n), np.zeros(n), x.get(), layer.mean_gpu.to_numpy(np.float32, (m,)),
                layer.rstd_gpu.to_numpy(np.float32, (m,)), "f32")


def _norm_grad(m, n, dtype, gap=0, want=("x", "g", "b"), in_place=False, affine=True):
    from tcbnn_amd import head
    r, x, gamma, _ = _norm_inputs(m, n, dtype, gap)
    if not affine:
        gamma = None
    gv = gamma.astype(np.float64) if affine else np.ones(n)
    dy = ho.Matrix(r.standard_normal((m, n)), dtype, gap)
    dyv = dy.values
    _, mean, rstd = ho.norm(x.values, 1.0, 0.0, EPS)
    mean, rstd = mean.astype(np.float32), rstd.astype(np.float32)
    dx, dg, db = dy if in_place else ho.Matrix(None, dtype, gap, m, n), ho.empty(n), ho.empty(n)
    layer = head.LayerNormLayerParam("norm", m, n, dtype, EPS)
    layer.initialize(gamma, None, x.view, mean_gpu=ho.vector(mean), rstd_gpu=ho.vector(rstd))
    layer.initialize_backward(dy.view, dx.view if "x" in want else None, dg if "g" in want else None, db if "b" in want else None)
    layer.backward()
    ho.sync()
    mean, rstd = mean.astype(np.float64)[:, None], rstd.astype(np.float64)[:, None]
    xh, g = (x.values - mean) * rstd, dyv * gv
    xerr = 3 * ho.U32 * np.abs(xh) + ho.U32 * np.abs(x.values) * rstd
    if "x" in want:
        mg, mgx = g.mean(1, keepdims=True), (g * xh).mean(1, keepdims=True)
        exact = (g - mg - xh * mgx) * rstd
        depth = (n / 64 + 24) * ho.U32
        e1 = depth * np.abs(g).mean(1, keepdims=True)
        e2 = depth * np.abs(g * xh).mean(1, keepdims=True) + (np.abs(g) * xerr).mean(1, keepdims=True)
        err = rstd * (e1 + np.abs(xh) * e2 + xerr * np.abs(mgx) + 6 * ho.U32 * (np.abs(g) + np.abs(mg) + np.abs(xh * mgx)))
        ho.check(dx.get(), exact, err + ho.U[dtype] * (np.abs(exact) + err) + ho.TINY[dtype], "grad_input")
    if "g" in want:
        err = (m + 2) * ho.U32 * np.abs(dyv * xh).sum(0) + (np.abs(dyv) * xerr).sum(0)
        ho.check(dg.to_numpy(np.float32, (n,)), (dyv * xh).sum(0), err, "grad_gamma")
    if "b" in want:
        ho.check(db.to_numpy(np.float32, (n,)), dyv.sum(0), m * ho.U32 * np.abs(dyv).sum(0), "grad_beta")
    layer.release()


@pytest.mark.parametrize("dtype", ho.DTYPES)
@pytest.mark.parametrize("m,n", NORM + [(2000, 24), (3001, 130), (600, 1000)])
def test_layernorm_grad(gpu, m, n, dtype):
    _norm_grad(m, n, dtype)
    _norm_grad(m, n, dtype, GAPS[dtype], affine=False)


@pytest.mark.parametrize("dtype", ho.DTYPES)
@pytest.mark.parametrize("m,n", [(5, 72), (130, 1001)])
def test_layernorm_grad_single_outputs_and_in_place(gpu, m, n, dtype):
    for want in (("x",), ("g",), ("b",), ("x", "b")):
        _norm_grad(m, n, dtype, want=want)
    _norm_grad(m, n, dtype, 8, in_place=True)


@pytest.mark.parametrize("dtype,n", [("f32", 8195), ("bf16", 16392)])
def test_layernorm_of_many_long_rows(gpu, dtype, n):
    """Rows that a workgroup's registers do not hold, more of them than workgroups run at a time."""
    from tcbnn_amd import head
    m = 1100
    r, x, gamma, beta = _norm_inputs(m, n, dtype, 0)
    layer = head.LayerNormLayerParam("norm", m, n, dtype, EPS).initialize(gamma, beta, x.view, output_gpu=x.view)
    want = x.values
    layer.forward()
    ho.sync()
    _check_norm(want, gamma.astype(np.float64), beta.astype(np.float64), x.get(), layer.mean_gpu.to_numpy(np.float32, (m,)),
                layer.rstd_gpu.to_numpy(np.float32, (m,)), dtype)
    layer.release()
    _norm_grad(m, n, dtype, in_place=True)


def test_layernorm_of_more_long_rows_than_a_launch_has(gpu):
    """2^22 workgroups of 1024 threads are more than a grid has: equal values become beta in every row, the last ones too."""
    import ctypes as C
    from tcbnn_amd import _lib, head
    m, n = (1 << 22) + 5, 8193
    free, total = C.c_size_t(0), C.c_size_t(0)
    _lib.hip.hipMemGetInfo(C.byref(free), C.byref(total))
    if free.value < 4 * m * n + (8 << 30):
        pytest.skip("needs %d GB of device memory" % (4 * m * n >> 30))
    x, beta = ho.DeviceBuffer(4 * m * n), np.arange(n, dtype=np.float32)
    x.fill(0x3c)
    layer = head.LayerNormLayerParam("norm", m, n, "f32", EPS).initialize(None, beta, x, output_gpu=x)
    layer.forward()
    ho.sync()
    value = np.uint32(0x3c3c3c3c).view(np.float32)
    for first in (0, 5, m // 2, m - 8):
        got = ho.DeviceView(x.ptr + 4 * first * n, 4 * 8 * n).to_numpy(np.float32, (8, n))
        # the mean's error beside the value, times rstd
        np.testing.assert_allclose(got, np.tile(beta, (8, 1)), rtol=2 * ho.U32, atol=(n / 64 + 24) * ho.U32 * value / np.sqrt(EPS))
    layer.release()
    x.free()


def test_layernorm_without_rows(gpu):
    from tcbnn_amd import head
    x, dg, db, one = ho.Matrix(None, "f32", 0, 0, 40), ho.empty(40), ho.empty(40), ho.empty(1)
    layer = head.LayerNormLayerParam("norm", 0, 40).initialize(None, None, x.view, output_gpu=x.view, mean_gpu=one, rstd_gpu=one)
    layer.initialize_backward(x.view, x.view, dg, db)
    layer.forward()
    layer.backward()
    ho.sync()
    assert not dg.to_numpy(np.float32, (40,)).any() and not db.to_numpy(np.float32, (40,)).any()


# --------------------------------------------------------------------------- log probabilities
# (rows, classes, top): one class; around a wavefront, a workgroup's share and several of them; few rows of many classes
# and many rows of few
LOGPROBS = [(3, 1, 1), (5, 2, 2), (700, 10, 5), (9, 63, 5), (4, 64, 64), (7, 65, 20), (33, 257, 8), (256, 1000, 5), (3, 1025, 32),
            (2, 4095, 64), (5, 4097, 0), (2, 8192, 5), (3, 16385, 20), (1, 32003, 20), (2, 50257, 1), (1, 131072, 20),
            (300, 2050, 3), (1, 262147, 64), (2, 24255, 9), (260, 32776, 7)]


def _logits(r, m, n, kind):
    x = 3.0 * r.standard_normal((m, n))
    if kind == "ties":
        x = np.round(x * 2) / 2
    elif kind == "equal":
        x[:] = np.round(x[:, :1], 1)
    elif kind == "sorted":
        x = np.sort(x, 1)
        x[::2] = x[::2, ::-1]
    elif kind == "cluster":  # the best classes lie side by side
        x[:, n // 3:n // 3 + 80] += 30.0
    elif kind == "stride":  # ... or a power of two apart
        x[:, ::64] += 30.0
    elif kind == "masked":
        x[r.random((m, n)) < 0.5] = -np.inf
        x[0] = -np.inf
        x[-1] = -np.inf
        x[-1, n // 2] = 0.25
    elif kind == "lowest":  # masks of the type's lowest value
        low = np.finfo(np.float16).min
        x[r.random((m, n)) < 0.7] = low
        x[0] = low
    elif kind == "special":
        x[0, n // 2] = np.nan
        x[m // 2, n - 1] = np.inf
        x[-1, 0] = -0.0
        x[-1, n - 1] = 0.0
    return x


def _logprobs(m, n, top, dtype, kind="plain", gap=0, stream=None):
    from tcbnn_amd import head
    r = rng(m, n, top, len(kind))
    x = ho.Matrix(_logits(r, m, n, kind), dtype, gap)
    t = r.integers(0, n, m).astype(np.int32)
    t[::5] = x.values[::5].argmax(1)
    t[3::7] = -1
    t[4::50] = n + 3
    layer = head.LogProbsLayerParam("logprobs", m, n, top, dtype).initialize(x.view, ho.vector(t, np.int32))
    layer.forward(stream)
    ho.sync()
    got = layer.download_output()
    xs = x.values
    want = [ho.logprobs(xs[i], int(t[i]), top) for i in range(m)]
    np.testing.assert_array_equal(got["rank"], [w[3] for w in want])
    if top:
        np.testing.assert_array_equal(got["top_index"], np.stack([w[4] for w in want]))
    # exp is good to 2 units of its result and 1.5 of its argument, terms of large arguments being small: |d| exp(d) < 0.4;
    # sums over at least 64 lanes; the logarithm, and roundings of the size of the largest logit
    big = np.array([np.abs(row[np.isfinite(row)]).max(initial=0.0) if row.max() < 100 else 0.0 for row in xs])
    depth = n / 64 + 24
    with np.errstate(invalid="ignore"):
        m_ = np.array([row.max() for row in xs])
    top_size = np.where(np.isfinite(m_), np.abs(np.where(np.isfinite(m_), m_, 0)), 0)
    lerr = (depth + 8) * ho.U32 + 4 * ho.U32 * (top_size + np.log(n) + 1)
    ho.check(got["logsumexp"], [w[2] for w in want], lerr, "logsumexp")
    lp = np.array([w[0] for w in want])
    ho.check(got["logprob"], lp, lerr + 2 * ho.U32 * (np.abs(np.where(np.isfinite(lp), lp, 0)) + top_size), "logprob")
    ent = np.array([w[1] for w in want])
    eerr = (2 * depth + 24) * ho.U32 * (np.log(n) + 2 + np.where(np.isfinite(ent), ent, 0))
    ho.check(got["entropy"], ent, eerr, "entropy")
    if top:
        lp = np.stack([w[5] for w in want])
        ho.check(got["top_logprob"], lp, lerr[:, None] + 2 * ho.U32 * (np.abs(np.where(np.isfinite(lp), lp, 0)) + top_size[:, None]),
                 "top_logprob")
    layer.release()


@pytest.mark.parametrize("dtype", ho.DTYPES)
@pytest.mark.parametrize("m,n,top", LOGPROBS)
def test_logprobs(gpu, m, n, top, dtype):
    _logprobs(m, n, top, dtype)


@pytest.mark.parametrize("dtype", ho.DTYPES)
@pytest.mark.parametrize("kind", ["ties", "equal", "sorted", "cluster", "stride", "masked", "lowest", "special"])
@pytest.mark.parametrize("m,n,top", [(4, 100, 64), (3, 1000, 20), (2, 4099, 64), (2, 24255, 33), (3, 33001, 33), (2, 140000, 64)])
def test_logprobs_of_rows_that_are_hard_to_rank(gpu, m, n, top, kind, dtype):
    _logprobs(m, n, top, dtype, kind, gap=GAPS[dtype] if n % 2 else 8)


# one wavefront a row (dealt, and in vectors), four, and rows in several chunks
SHAPES = [(4, 100, 20), (3, 1000, 20), (2, 4099, 33), (2, 24255, 33), (3, 33001, 20), (2, 140000, 64)]


def _about_the_largest(x, t, top):
    """ho.logprobs() of a row of finite logits, with log probabilities as (x - m) - log sum: x - logsumexp loses the sum's
    logarithm in any type once the logits are large enough."""
    _, _, _, rank, best, _ = ho.logprobs(x, t, top)
    d = x - x.max()
    log_sum = np.log(np.exp(d).sum())
    p = np.exp(d - log_sum)
    lp = d - log_sum
    return lp[t], -(p * np.where(p > 0, lp, 0.0)).sum(), x.max() + log_sum, rank, best, lp[best]


def _against_definition(x, t, top, dtype):
    """forward() of rows given as a Matrix, with tolerances that do not grow with the logits: exp and log are good to two units, the
    argument of exp adds 1.5 of its size, whose mean under the distribution is below log n; sums over at least 64 lanes; x - m
    and a log probability are rounded once each.  A logsumexp's own rounding is of its size."""
    from tcbnn_amd import head
    m, n = x.shape
    layer = head.LogProbsLayerParam("logprobs", m, n, top, dtype).initialize(x.view, ho.vector(t, np.int32))
    layer.forward()
    ho.sync()
    got = layer.download_output()
    want = [_about_the_largest(x.values[i], int(t[i]), top) for i in range(m)]
    np.testing.assert_array_equal(got["rank"], [w[3] for w in want])
    np.testing.assert_array_equal(got["top_index"], np.stack([w[4] for w in want]))
    depth, log_n = n / 64 + 24, np.log(n)
    base = ho.U32 * (depth + 8 + 4 * log_n)
    lp, lse, ent, best = (np.array([w[k] for w in want]) for k in (0, 2, 1, 5))
    ho.check(got["logprob"], lp, base + 2 * ho.U32 * np.abs(lp), "logprob")
    ho.check(got["top_logprob"], best, base + 2 * ho.U32 * np.abs(best), "top_logprob")
    ho.check(got["logsumexp"], lse, base + 1.01 * ho.U32 * np.abs(lse), "logsumexp")
    ho.check(got["entropy"], ent, (2 * depth + 24) * ho.U32 * (log_n + 2 + ent), "entropy")
    layer.release()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("m,n,top", SHAPES)
def test_logprobs_far_from_zero(gpu, m, n, top, dtype):
    """Finite logits about any value: spread as far as the type's neighbours are there, and all equal."""
    r = rng(m, n, 21)
    for about in (1e5, 1e6, -1e6, 1e7, 1e9, -1e9, 1e20, -1e30, 1e37, 3e38):
        v = about + 3.0 * r.standard_normal((m, n))
        v[-1] = about
        v[0] *= 1.0 - 2.0 ** -8 * r.integers(0, 3, n)
        _against_definition(ho.Matrix(v, dtype), r.integers(0, n, m).astype(np.int32), top, dtype)


@pytest.mark.parametrize("dtype", ho.DTYPES)
@pytest.mark.parametrize("m,n,top", SHAPES)
def test_logprobs_at_ordinary_offsets(gpu, m, n, top, dtype):
    """Entropies and log probabilities as good about 60000 as about 0."""
    r = rng(m, n, 23)
    for about in (-30.0, 100.0, -1000.0, 3000.0, 20000.0, -60000.0, 60000.0):
        _against_definition(ho.Matrix(about + 2.5 * r.standard_normal((m, n)), dtype), r.integers(0, n, m).astype(np.int32), top, dtype)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("value", [-1e9, -1e10, -1e30, "lowest"])
@pytest.mark.parametrize("m,n,top", SHAPES)
def test_logprobs_of_finite_masks(gpu, m, n, top, value, dtype):
    """A finite value in the place of forbidden classes: behind the allowed ones (whole wavefronts' shares and chunks), before them,
    in all places but one, in all."""
    if value == "lowest":
        value = {"f32": -3.4028234663852886e38, "bf16": -3.3895313892515355e38}[dtype]
    r = rng(m, n, 22)
    for first, last in ((n // 3, n), (0, n - n // 5), (0, n), (n // 2 + 1, n)):
        v = 3.0 * r.standard_normal((m, n))
        v[:, first:last] = value
        if last - first < n // 2:
            v[:, :first - 1] = value
        t = r.integers(0, n, m).astype(np.int32)
        t[0] = first - 1 if first else (last if last < n else 0)
        _against_definition(ho.Matrix(v, dtype), t, top, dtype)


@pytest.mark.parametrize("dtype", ho.DTYPES)
@pytest.mark.parametrize("m,n,top", SHAPES)
def test_logprobs_of_negative_zeros(gpu, m, n, top, dtype):
    """-0 and +0 are equal logits: a target that holds either has the rank that its index among them says, and is where the best
    classes say."""
    from tcbnn_amd import head
    r = rng(m, n, 24)
    for share in (0.0, 0.5, 1.0):  # of -0 among the classes besides the target
        v = np.where(r.random((m, n)) < share, -0.0, 0.0)
        v[1, r.integers(0, n, n // 4)] = -1.0
        v[-1, r.integers(0, n, 3)] = 1.0
        for sign in (-0.0, 0.0):
            for at in (0, 5, n // 2, n - 1, n // 3 + 1):
                t = np.full(m, at, np.int32)
                w = v.copy()
                w[:, at] = sign
                x = ho.Matrix(w, dtype)
                layer = head.LogProbsLayerParam("logprobs", m, n, top, dtype).initialize(x.view, ho.vector(t, np.int32))
                layer.forward()
                ho.sync()
                got = layer.download_output()
                want = [ho.logprobs(row, at, top) for row in x.values]
                np.testing.assert_array_equal(got["rank"], [a[3] for a in want])
                np.testing.assert_array_equal(got["top_index"], np.stack([a[4] for a in want]))
                for i in range(m):
                    if got["rank"][i] < top:
                        assert got["top_index"][i, got["rank"][i]] == at
                layer.release()


@pytest.mark.parametrize("dtype", ho.DTYPES)
@pytest.mark.parametrize("m,n,top", SHAPES + [(2, 1, 1), (3, 64, 64), (2, 70000, 20)])
def test_logprobs_of_nans_in_first_places(gpu, m, n, top, dtype):
    """NaN goes before every number wherever it is: in class 0, in the first class of a wavefront's share or a chunk, in all."""
    from tcbnn_amd import head
    r = rng(m, n, 25)
    for places in (slice(0, 1), slice(0, n, 4096), slice(0, n, 32768), slice(n - 1, n), slice(0, n)):
        v = r.standard_normal((m, n))
        v[:, places] = np.nan
        t = np.zeros(m, np.int32)
        t[-1] = n - 1
        x = ho.Matrix(v, dtype)
        layer = head.LogProbsLayerParam("logprobs", m, n, top, dtype).initialize(x.view, ho.vector(t, np.int32))
        layer.forward()
        ho.sync()
        got = layer.download_output()
        want = [ho.logprobs(x.values[i], int(t[i]), top) for i in range(m)]
        np.testing.assert_array_equal(got["rank"], [w[3] for w in want])
        np.testing.assert_array_equal(got["top_index"], np.stack([w[4] for w in want]))
        assert np.isnan(got["logprob"]).all() and np.isnan(got["top_logprob"]).all() and np.isnan(got["entropy"]).all()
        layer.release()


def test_logprobs_outputs_are_optional(gpu):
    """What is not asked for is not needed: entropy alone, the best classes alone."""
    import ctypes as C
    from tcbnn_amd import _lib
    r = rng(5)
    x = ho.Matrix(r.standard_normal((4, 300)), "f32")
    want = [ho.logprobs(v, -1, 3) for v in x.values]
    entropy, index = ho.empty(4), ho.empty(12, np.int32)
    ws_bytes = _lib.lib.tcbnn_logprobs_workspace_bytes(4, 300, 3, 0)
    ws = ho.DeviceBuffer(ws_bytes)
    d = _lib.LogProbsDesc(logits=x.view.ptr, entropy=entropy.ptr, rows=4, classes=300, dtype=0, workspace=ws.ptr,
                          workspace_bytes=ws_bytes)
    _lib.check(_lib.lib.tcbnn_logprobs_forward(C.byref(d), None))
    d = _lib.LogProbsDesc(logits=x.view.ptr, top_index=index.ptr, rows=4, classes=300, top=3, dtype=0, workspace=ws.ptr,
                          workspace_bytes=ws_bytes)
    _lib.check(_lib.lib.tcbnn_logprobs_forward(C.byref(d), None))
    ho.sync()
    ho.check(entropy.to_numpy(np.float32, (4,)), [w[1] for w in want], 1e-5)
    np.testing.assert_array_equal(index.to_numpy(np.int32, (4, 3)), np.stack([w[4] for w in want]))


def _logprobs_grad(m, n, dtype, kind="plain", gap=0, entropy=True, logprob=True, in_place=False):
    from tcbnn_amd import head
    r = rng(m, n, len(kind), 2)
    x = ho.Matrix(_logits(r, m, n, kind), dtype, gap)
    xs = x.values
    t = r.integers(0, n, m).astype(np.int32)
    t[3::7] = -1
    t[4::50] = n
    with np.errstate(invalid="ignore", divide="ignore"):
        rows = [ho.logprobs(v, -1, 0) for v in xs]
    lse, ent = np.array([w[2] for w in rows], np.float32), np.array([w[1] for w in rows], np.float32)
    g, ge = r.standard_normal(m).astype(np.float32), r.standard_normal(m).astype(np.float32)
    dx = x if in_place else ho.Matrix(None, dtype, gap, m, n)
    layer = head.LogProbsLayerParam("logprobs", m, n, 0, dtype)
    layer.initialize(x.view, ho.vector(t, np.int32), logsumexp_gpu=ho.vector(lse), entropy_gpu=ho.vector(ent))
    layer.initialize_backward(ho.vector(g) if logprob else None, ho.vector(ge) if entropy else None, dx.view)
    layer.backward()
    ho.sync()
    got = dx.get()
    for i in range(m):
        gi = 0.0 if not logprob or t[i] < 0 else (np.nan if t[i] >= n else float(g[i]))
        gei = float(ge[i]) if entropy else 0.0
        if lse[i] == -np.inf:
            want, err = np.full(n, np.nan if np.isnan(gi) else 0.0), 0.0
        else:
            with np.errstate(invalid="ignore"):
                lp = xs[i] - np.float64(lse[i])
                p = np.exp(lp)
                hot = np.zeros(n)
                if 0 <= t[i] < n:
                    hot[t[i]] = 1.0
                l0 = np.where(p > 0, lp, 0.0)
                want = gi * (hot - p) - gei * p * (l0 + ent[i])
                # exp: a rounding of its argument's size, and its own
                perr = p * ho.U32 * (4 + 3 * np.abs(l0) + 2 * np.abs(lse[i]))
                err = (abs(gi) * (perr + 3 * ho.U32 * (hot + p)) + abs(gei) * (perr * np.abs(l0 + ent[i])
                       + p * ho.U32 * (6 * np.abs(l0) + 4 * abs(ent[i]) + 2 * np.abs(lse[i]))))
        with np.errstate(invalid="ignore"):
            tol = err + ho.U[dtype] * (np.abs(want) + err) + ho.TINY[dtype]
        ho.check(got[i], want, tol, "row %d" % i)
    layer.release()


@pytest.mark.parametrize("dtype", ho.DTYPES)
@pytest.mark.parametrize("m,n", [(3, 1), (60, 10), (9, 64), (5, 1000), (3, 1025), (2, 4097), (2, 32003), (1, 131072)])
def test_logprobs_grad(gpu, m, n, dtype):
    _logprobs_grad(m, n, dtype)
    _logprobs_grad(m, n, dtype, gap=GAPS[dtype], entropy=False)
    _logprobs_grad(m, n, dtype, gap=8, logprob=False)
    _logprobs_grad(m, n, dtype, in_place=True)


@pytest.mark.parametrize("dtype", ho.DTYPES)
@pytest.mark.parametrize("kind", ["equal", "masked", "lowest", "special"])
@pytest.mark.parametrize("m,n", [(4, 100), (3, 2051)])
def test_logprobs_grad_of_special_rows(gpu, m, n, kind, dtype):
    _logprobs_grad(m, n, dtype, kind)


def test_logprobs_of_more_rows_than_a_launch_has(gpu):
    """A grid has fewer than 2^32 threads: 2^26 rows of few classes forward, 2^24 backward.  The rows repeat with an odd period."""
    from tcbnn_amd import head
    n, period = 2, 4099
    r = rng(31)
    values = r.standard_normal((period, n)).astype(np.float16)
    targets, g = r.integers(-1, n, period).astype(np.int32), r.standard_normal(period).astype(np.float32)
    want = [ho.logprobs(v.astype(np.float64), int(t), 1) for v, t in zip(values, targets)]

    def rows(a, m):
        return ho.DeviceBuffer.from_numpy(np.resize(a, (m,) + a.shape[1:]))

    def repeats(got, a, tol):
        wide = np.resize(np.asarray(a, np.float32), (got.shape[0],) + np.shape(a)[1:])
        worst = np.abs(got.astype(np.float32) - wide).max()
        assert worst <= tol, worst

    m = (1 << 26) + 77
    layer = head.LogProbsLayerParam("logprobs", m, n, 1, "f16").initialize(rows(values, m), rows(targets, m))
    layer.forward()
    ho.sync()
    for name, k in (("logprob", 0), ("entropy", 1), ("logsumexp", 2), ("rank", 3), ("top_index", 4), ("top_logprob", 5)):
        buf = getattr(layer, name + "_gpu")
        whole = name in ("rank", "top_index")
        got = buf.to_numpy(np.int32 if whole else np.float32, (m,))
        repeats(got, [np.ravel(w[k])[0] for w in want], 0 if whole else 1e-5)
    layer.release()
    m = (1 << 24) + 77
    layer = head.LogProbsLayerParam("logprobs", m, n, 0, "f16").initialize(rows(values, m), rows(targets, m))
    dx = ho.DeviceBuffer(2 * m * n)
    dx.fill(0x7f)
    layer.initialize_backward(rows(g, m), None, dx)
    layer.forward()
    layer.backward()
    ho.sync()
    lse = np.array([w[2] for w in want])
    hot = (np.arange(n) == targets[:, None]) - np.exp(values.astype(np.float64) - lse[:, None])
    repeats(dx.to_numpy(np.float16, (m, n)), np.where(targets[:, None] < 0, 0.0, g[:, None] * hot), 2 * ho.U["f16"] * 4 + 1e-5)
    layer.release()


# --------------------------------------------------------------------------- gradients against differences
def _slope_along(f, x, v):
    h = 1e-5
    return (f(x + h * v) - f(x - h * v)) / (2 * h)


def test_gradients_against_differences(gpu):
    """Norm -> linear (GELU, residual) -> log probabilities in fp32 on the GPU, forward and backward through the layers,
    against central differences of the definition in 64 bits along random directions."""
    from tcbnn_amd import head
    m, k, n = 21, 40, 30
    r = rng(11)
    x, wt = r.standard_normal((m, k)), r.standard_normal((n, k)) / np.sqrt(k)
    gamma, beta, b = 1 + 0.1 * r.standard_normal(k), 0.1 * r.standard_normal(k), 0.1 * r.standard_normal(n)
    res = r.standard_normal((m, n))
    t = r.integers(0, n, m).astype(np.int32)
    g, ge = r.standard_normal(m), r.standard_normal(m)
    x, wt, gamma, beta, b, res, g, ge = (a.astype(np.float32).astype(np.float64) for a in (x, wt, gamma, beta, b, res, g, ge))

    def loss(x, gamma, beta, wt, b, res):
        y, _, _ = ho.norm(x, gamma, beta, EPS)
        z = ho.act("gelu", y @ wt.T + b) + res
        rows = [ho.logprobs(z[i], int(t[i]), 0) for i in range(m)]
        return sum(g[i] * rows[i][0] + ge[i] * rows[i][1] for i in range(m))

    mx = {name: ho.Matrix(a, "f32") for name, a in dict(x=x, w=wt, res=res).items()}
    out = {name: ho.Matrix(None, "f32", 0, *s) for name, s in dict(y=(m, k), z=(m, n), dz=(m, n), dy=(m, k), dx=(m, k), dw=(n, k)).items()}
    vec = {name: ho.empty(s) for name, s in dict(dgamma=k, dbeta=k, db=n).items()}
    norm = head.LayerNormLayerParam("norm", m, k).initialize(gamma, beta, mx["x"].view, output_gpu=out["y"].view)
    lin = head.LinearLayerParam("linear", m, k, n, activation="gelu").initialize(
        mx["w"].view, b, out["y"].view, residual_gpu=mx["res"].view, output_gpu=out["z"].view, save_preact=True)
    lps = head.LogProbsLayerParam("logprobs", m, n).initialize(out["z"].view, ho.vector(t, np.int32))
    lps.initialize_backward(ho.vector(g), ho.vector(ge), out["dz"].view)
    lin.initialize_backward(out["dz"].view, out["dy"].view, out["dw"].view, vec["db"])
    norm.initialize_backward(out["dy"].view, out["dx"].view, vec["dgamma"], vec["dbeta"])
    for layer in (norm, lin, lps):
        layer.forward()
    for layer in (lps, lin, norm):
        layer.backward()
    ho.sync()
    args = dict(x=x, gamma=gamma, beta=beta, wt=wt, b=b, res=res)
    grads = dict(x=out["dx"].get(), gamma=vec["dgamma"].to_numpy(np.float32, (k,)), beta=vec["dbeta"].to_numpy(np.float32, (k,)),
                 wt=out["dw"].get(), b=vec["db"].to_numpy(np.float32, (n,)), res=out["dz"].get())
    for name, grad in grads.items():
        for _ in range(3):
            v = r.standard_normal(args[name].shape)
            want = _slope_along(lambda a: loss(**{**args, name: a}), args[name], v)
            # a few hundred fp32 roundings of terms of the gradient's own size
            assert abs((grad * v).sum() - want) <= 200 * ho.U32 * np.abs(grad * v).sum() + 1e-6, name
    for layer in (norm, lin, lps):
        layer.release()
