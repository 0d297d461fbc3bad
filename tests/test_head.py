"""The float head without a GPU: what its entry points refuse (nothing is launched), what its layers refuse, the rounding of
parameters, and the definitions that the GPU tests compare with, against differences."""
import ctypes as C

import numpy as np
import pytest

from tests import headops as ho

EINVAL, ENULL = -1, -2
P = 0x1000  # a pointer that no refused call follows


def _lib():
    from tcbnn_amd import _lib
    return _lib


def _linear(**kw):
    d = dict(input=P, weight=P, output=P, rows=4, in_features=8, out_features=8, dtype=1, activation=0)
    return "tcbnn_linear_forward", _lib().LinearDesc(**{**d, **kw})


def _linear_grad(**kw):
    d = dict(input=P, weight=P, preact=P, grad_output=P, grad_input=P, grad_weight=P, grad_bias=P, rows=4, in_features=8,
             out_features=8, dtype=1, activation=2, workspace=P, workspace_bytes=1 << 30)
    return "tcbnn_linear_backward", _lib().LinearGradDesc(**{**d, **kw})


def _norm(**kw):
    d = dict(input=P, output=P, rows=4, features=8, dtype=1, eps=1e-5)
    return "tcbnn_layernorm_forward", _lib().LayerNormDesc(**{**d, **kw})


def _norm_grad(**kw):
    d = dict(input=P, mean=P, rstd=P, grad_output=P, grad_input=P, grad_gamma=P, rows=4, features=8, dtype=1, workspace=P,
             workspace_bytes=1 << 30)
    return "tcbnn_layernorm_backward", _lib().LayerNormGradDesc(**{**d, **kw})


def _logprobs(**kw):
    d = dict(logits=P, targets=P, logprob=P, top_index=P, rows=4, classes=80, top=5, dtype=1, workspace=P, workspace_bytes=1 << 30)
    return "tcbnn_logprobs_forward", _lib().LogProbsDesc(**{**d, **kw})


def _logprobs_grad(**kw):
    d = dict(logits=P, targets=P, logsumexp=P, entropy=P, grad_logprob=P, grad_entropy=P, grad_logits=P, rows=4, classes=80, dtype=1)
    return "tcbnn_logprobs_backward", _lib().LogProbsGradDesc(**{**d, **kw})


@pytest.mark.parametrize("make,change,code,message", [
    (_linear, dict(dtype=3), EINVAL, "dtype"), (_linear, dict(dtype=-1), EINVAL, "dtype"),
    (_linear, dict(activation=4), EINVAL, "activation"), (_linear, dict(rows=-1), EINVAL, "shape"),
    (_linear, dict(in_features=0), EINVAL, "shape"), (_linear, dict(out_features=0), EINVAL, "shape"),
    (_linear, dict(in_features=(1 << 20) + 1), EINVAL, "inputs"), (_linear, dict(input_ld=7), EINVAL, "overlap"),
    (_linear, dict(weight_ld=7), EINVAL, "overlap"), (_linear, dict(output_ld=7), EINVAL, "overlap"),
    (_linear, dict(residual_ld=-8), EINVAL, "overlap"), (_linear, dict(preact_ld=1), EINVAL, "overlap"),
    (_linear, dict(input=0), ENULL, "input"), (_linear, dict(weight=0), ENULL, "weight"), (_linear, dict(output=0), ENULL, "output"),
    (_linear, dict(residual=P, residual_ld=16), EINVAL, "stride"),
    (_linear_grad, dict(dtype=9), EINVAL, "dtype"), (_linear_grad, dict(activation=-1), EINVAL, "activation"),
    (_linear_grad, dict(rows=-4), EINVAL, "shape"), (_linear_grad, dict(grad_output=0), ENULL, "grad_output"),
    (_linear_grad, dict(preact=0), ENULL, "preact"), (_linear_grad, dict(input=0), ENULL, "input"),
    (_linear_grad, dict(weight=0), ENULL, "weight"), (_linear_grad, dict(workspace=0), ENULL, "workspace"),
    (_linear_grad, dict(workspace_bytes=1), EINVAL, "workspace"), (_linear_grad, dict(grad_weight_ld=4), EINVAL, "overlap"),
    (_norm, dict(dtype=3), EINVAL, "dtype"), (_norm, dict(features=0), EINVAL, "shape"), (_norm, dict(features=65537), EINVAL, "features"),
    (_norm, dict(eps=-1.0), EINVAL, "eps"), (_norm, dict(eps=float("nan")), EINVAL, "eps"), (_norm, dict(input=0), ENULL, "input"),
    (_norm, dict(output=0), ENULL, "output"), (_norm, dict(input_ld=7), EINVAL, "overlap"),
    (_norm, dict(output_ld=16), EINVAL, "stride"),
    (_norm_grad, dict(rows=-1), EINVAL, "shape"), (_norm_grad, dict(mean=0), ENULL, "mean"), (_norm_grad, dict(rstd=0), ENULL, "rstd"),
    (_norm_grad, dict(input=0), ENULL, "input"), (_norm_grad, dict(grad_output=0), ENULL, "grad_output"),
    (_norm_grad, dict(grad_input_ld=3), EINVAL, "overlap"), (_norm_grad, dict(features=1 << 17), EINVAL, "features"),
    (_logprobs, dict(classes=0), EINVAL, "shape"), (_logprobs, dict(top=65), EINVAL, "top"), (_logprobs, dict(top=-1), EINVAL, "top"),
    (_logprobs, dict(classes=4), EINVAL, "top"), (_logprobs, dict(logits=0), ENULL, "logits"),
    (_logprobs, dict(targets=0), ENULL, "targets"), (_logprobs, dict(logprob=0, rank=P, targets=0), ENULL, "targets"),
    (_logprobs, dict(logits_ld=79), EINVAL, "overlap"), (_logprobs, dict(dtype=4), EINVAL, "dtype"),
    (_logprobs_grad, dict(classes=-2), EINVAL, "shape"), (_logprobs_grad, dict(logits=0), ENULL, "logits"),
    (_logprobs_grad, dict(logsumexp=0), ENULL, "logsumexp"), (_logprobs_grad, dict(entropy=0), ENULL, "entropy"),
    (_logprobs_grad, dict(targets=0), ENULL, "targets"), (_logprobs_grad, dict(grad_logits=0), ENULL, "grad_logits"),
    (_logprobs_grad, dict(grad_logits=P, grad_logits_ld=96), EINVAL, "stride"),
])
def test_refusals(make, change, code, message):
    if make is _linear and "residual" in change:
        change = dict(change, output=P)
    if make is _norm and "output_ld" in change:
        change = dict(change, output=P)
    entry, d = make(**change)
    lib = _lib().lib
    assert getattr(lib, entry)(C.byref(d), None) == code
    assert message in lib.tcbnn_last_error().decode()


@pytest.mark.parametrize("change", [dict(), dict(activation=0), dict(activation=0, grad_bias=0), dict(activation=0, grad_bias=0, grad_weight=0),
                                    dict(activation=0, grad_bias=0, grad_input=0)])
def test_linear_gradients_need_their_workspace(change):
    """The whole of it, whichever gradients are asked for: how a sum is split does not go by what is there."""
    lib = _lib().lib
    need = lib.tcbnn_linear_grad_workspace_bytes(4, 8, 8, 1)
    for workspace, code in ((dict(workspace=0), ENULL), (dict(workspace_bytes=need - 1), EINVAL), (dict(workspace=P + 4), EINVAL)):
        entry, d = _linear_grad(**{**change, **workspace})
        assert getattr(lib, entry)(C.byref(d), None) == code
        assert "workspace" in lib.tcbnn_last_error().decode()


@pytest.mark.parametrize("rows", [(1 << 31) - 1, (1 << 31) - 600, (1 << 31) - (1 << 22) + 1])
def test_linear_refuses_rows_that_its_sums_do_not_count(rows):
    """The gradient of the weight sums over the rows, a step at a time past the last one: within 32 bits."""
    lib = _lib().lib
    for entry, d in (_linear(rows=rows), _linear_grad(rows=rows, workspace_bytes=1 << 62), _linear_grad(rows=rows, workspace_bytes=1 << 62, grad_input=0)):
        assert getattr(lib, entry)(C.byref(d), None) == EINVAL
        assert "rows" in lib.tcbnn_last_error().decode()
    d = _linear(rows=rows)[1]
    assert lib.tcbnn_linear_kernel_name(C.byref(d), C.create_string_buffer(160), 160) == EINVAL
    assert lib.tcbnn_linear_workspace_bytes(rows, 8, 8, 1) == lib.tcbnn_linear_grad_workspace_bytes(rows, 8, 8, 1) == 0


def test_no_rows_and_null_descriptors():
    lib = _lib().lib
    for entry, d in (_linear(rows=0, input=0, output=0), _norm(rows=0, input=0, output=0), _logprobs(rows=0, logits=0),
                     _logprobs_grad(rows=0, logits=0)):
        assert getattr(lib, entry)(C.byref(d), None) == 0
    for entry in ("tcbnn_linear_forward", "tcbnn_linear_backward", "tcbnn_layernorm_forward", "tcbnn_layernorm_backward",
                  "tcbnn_logprobs_forward", "tcbnn_logprobs_backward"):
        assert getattr(lib, entry)(None, None) == ENULL


def test_workspaces_of_refused_sizes_are_empty():
    lib = _lib().lib
    assert lib.tcbnn_linear_workspace_bytes(0, 8, 8, 0) == lib.tcbnn_linear_workspace_bytes(4, -1, 8, 0) == 0
    assert lib.tcbnn_linear_grad_workspace_bytes(4, 8, 0, 0) == lib.tcbnn_linear_grad_workspace_bytes(4, 8, 8, 7) == 0
    assert lib.tcbnn_layernorm_grad_workspace_bytes(0, 8) == lib.tcbnn_layernorm_grad_workspace_bytes(4, -8) == 0
    assert lib.tcbnn_logprobs_workspace_bytes(-1, 8, 0, 0) == lib.tcbnn_logprobs_workspace_bytes(4, 8, 99, 0) == 0


def test_kernel_names():
    """The kernel of a forward call by sizes and alignment; a workspace lets few tiles share a long sum; nothing is followed."""
    lib = _lib().lib

    def name(**kw):
        d = _linear(**{**dict(rows=64, in_features=16384, out_features=64), **kw})[1]
        buf = C.create_string_buffer(160)
        assert lib.tcbnn_linear_kernel_name(C.byref(d), buf, 160) == 0
        return buf.value.decode()

    need = lib.tcbnn_linear_workspace_bytes(64, 16384, 64, 1)
    assert need > 0 and "join" in name(workspace=P, workspace_bytes=need)
    assert "join" not in name() and "join" not in name(workspace=P, workspace_bytes=16)
    assert name(rows=16, in_features=1024) == "few_rows_kernel<__bf16, 8>" and name(rows=1, dtype=0, in_features=256) == "few_rows_kernel<float, 8>"
    assert name(rows=3, in_features=264, out_features=16408) == "few_rows_kernel<__bf16, 2>" and "32, 32" in name(rows=17, in_features=1024)
    assert "few" in name(rows=1) and "join" in name(rows=1, workspace=P, workspace_bytes=need)
    assert "(Access)0" in name() and "(Access)1" in name(input=P + 2) and "(Access)1" in name(input_ld=16387)
    assert "(Access)2" in name(in_features=5) and "(Access)2" in name(weight_ld=1 << 24)
    assert "256, 256" in name(rows=8192, in_features=4096, out_features=4096)
    d = _linear(rows=-1)[1]
    assert lib.tcbnn_linear_kernel_name(C.byref(d), C.create_string_buffer(8), 8) == EINVAL
    assert lib.tcbnn_linear_kernel_name(None, C.create_string_buffer(8), 8) == ENULL


def test_kernel_name_of_a_split_sum_of_far_rows():
    """Rows too far apart for a tile's 32-bit offsets: a long sum of few tiles is split, and joined, there too."""
    lib = _lib().lib
    need = lib.tcbnn_linear_workspace_bytes(64, 16384, 64, 1)
    buf = C.create_string_buffer(160)
    for workspace, joined in ((need, True), (0, False)):
        d = _linear(rows=64, in_features=16384, out_features=64, weight_ld=1 << 24, workspace=P if workspace else 0, workspace_bytes=workspace)[1]
        assert lib.tcbnn_linear_kernel_name(C.byref(d), buf, 160) == 0
        assert "(Access)2" in buf.value.decode() and ("product_join_kernel" in buf.value.decode()) == joined


def test_layers_refuse():
    from tcbnn_amd import head
    from tcbnn_amd.device import DeviceView
    E = _lib().TcbnnError
    buf = DeviceView(P, 4 * 64)
    with pytest.raises(E, match="dtype"):
        head.LinearLayerParam("l", 4, 8, 8, "f64")
    with pytest.raises(E, match="activation"):
        head.LinearLayerParam("l", 4, 8, 8, "f32", "tanh")
    with pytest.raises(E, match="NULL pointer"):
        head.LinearLayerParam("l", 4, 8, 8).initialize(buf, None, None, output_gpu=buf)
    with pytest.raises(E, match="input holds"):
        head.LinearLayerParam("l", 9, 8, 8).initialize(buf, None, buf, output_gpu=buf)
    with pytest.raises(E, match="weight holds"):
        head.LinearLayerParam("l", 1, 8, 9).initialize(buf, None, buf, output_gpu=buf)
    with pytest.raises(E, match="preact"):
        head.LinearLayerParam("l", 1, 8, 8, activation="silu").initialize(buf, None, buf, output_gpu=buf).initialize_backward(buf)
    with pytest.raises(E, match="not initialized"):
        head.LayerNormLayerParam("n", 4, 8).forward()
    with pytest.raises(E, match="gamma holds"):
        head.LayerNormLayerParam("n", 1, 64).initialize(DeviceView(P, 60), None, buf, output_gpu=buf)
    with pytest.raises(E, match="targets"):
        head.LogProbsLayerParam("p", 4, 8).initialize(buf, entropy_gpu=buf, logsumexp_gpu=buf).initialize_backward(buf, None, buf)


def test_views_of_tensors():
    torch = pytest.importorskip("torch")
    from tcbnn_amd.device import DeviceView
    wide = torch.zeros((5, 12))
    v = DeviceView.of(wide[:, 2:9])
    assert (v.ptr, v.ld, v.nbytes) == (wide.data_ptr() + 8, 12, 4 * 35)
    assert DeviceView.of(wide[1]).ld == 0 and DeviceView.of(wide[:1, :7]).ld == 0
    for bad in (wide.t(), wide[:, ::2], wide.reshape(5, 3, 4)):
        with pytest.raises(_lib().TcbnnError):
            DeviceView.of(bad)


def test_views_of_broadcast_tensors():
    """Rows that share memory are fewer bytes than a layer would read or write."""
    torch = pytest.importorskip("torch")
    from tcbnn_amd.device import DeviceView
    row = torch.zeros(8)
    for bad in (row.expand(1000, 8), row[:1].expand(4, 1), torch.zeros((40,)).as_strided((5, 8), (4, 1)), row[:1].expand(8), torch.zeros(())):
        with pytest.raises(_lib().TcbnnError):
            DeviceView.of(bad)
    assert DeviceView.of(row.expand(1, 8)).nbytes == 32 and DeviceView.of(torch.zeros((0, 8))).nbytes == 0


def test_layers_refuse_other_element_types():
    """A view of a tensor knows its type: enough bytes of another one are not what a layer reads."""
    torch = pytest.importorskip("torch")
    from tcbnn_amd import head
    from tcbnn_amd.device import DeviceView
    E = _lib().TcbnnError

    def view(dtype, *shape):
        v = DeviceView.of(torch.zeros(shape, dtype=dtype))
        return DeviceView(P, v.nbytes, v.ld, dtype=v.dtype)

    f32, bf16, raw = view(torch.float32, 8, 8), view(torch.bfloat16, 8, 8), DeviceView(P, 256)
    assert (f32.dtype, bf16.dtype, view(torch.float16, 1).dtype, view(torch.int32, 1).dtype, raw.dtype) == ("f32", "bf16", "f16", "i32", None)
    with pytest.raises(E, match="input.*f32.*bf16"):
        head.LinearLayerParam("l", 8, 8, 8, "bf16").initialize(bf16, None, f32, output_gpu=bf16)
    with pytest.raises(E, match="weight"):
        head.LinearLayerParam("l", 8, 8, 8, "f32").initialize(view(torch.float64, 8, 8), None, f32, output_gpu=f32)
    with pytest.raises(E, match="bias"):
        head.LinearLayerParam("l", 8, 8, 8, "bf16").initialize(bf16, view(torch.bfloat16, 16), bf16, output_gpu=bf16)
    with pytest.raises(E, match="gamma"):
        head.LayerNormLayerParam("n", 8, 8, "f16").initialize(view(torch.float16, 16), None, view(torch.float16, 8, 8), output_gpu=raw)
    lp = head.LogProbsLayerParam("p", 8, 8)
    lp._buffer = lambda nbytes: DeviceView(P, nbytes)
    with pytest.raises(E, match="targets.*int64.*i32"):
        lp.initialize(f32, view(torch.int64, 8))
    with pytest.raises(E, match="rank"):
        lp.initialize(f32, view(torch.int32, 8), rank_gpu=view(torch.float32, 8))
    lp.initialize(f32, view(torch.int32, 8), rank_gpu=view(torch.int32, 8), entropy_gpu=view(torch.float32, 8))
    with pytest.raises(E, match="grad_logits"):
        lp.initialize_backward(raw, None, view(torch.float64, 8, 8))
    linear = head.LinearLayerParam("l", 8, 8, 8, "f32")  # (what does not say its type is taken at its size, as before)
    linear.initialize(raw, raw, raw, output_gpu=f32)


def test_layers_refuse_host_tensors():
    """A kernel does not follow a pointer into pageable host memory."""
    torch = pytest.importorskip("torch")
    from tcbnn_amd import head
    from tcbnn_amd.device import DeviceView
    E = _lib().TcbnnError
    buf, host = DeviceView(P, 256), DeviceView.of(torch.zeros(8, 8))
    assert host.on_host and not buf.on_host
    with pytest.raises(E, match="input.*host"):
        head.LinearLayerParam("l", 8, 8, 8).initialize(buf, None, host, output_gpu=buf)
    with pytest.raises(E, match="bias.*host"):
        head.LinearLayerParam("l", 8, 8, 8).initialize(buf, DeviceView.of(torch.zeros(8)), buf, output_gpu=buf)
    with pytest.raises(E, match="grad_output.*host"):
        head.LinearLayerParam("l", 8, 8, 8).initialize(buf, None, buf, output_gpu=buf).initialize_backward(host)


def test_layers_refuse_rows_that_are_not_there():
    """Rows some elements apart: as many, as long as a layer has, in memory that holds them; vectors without gaps."""
    torch = pytest.importorskip("torch")
    from tcbnn_amd import head
    from tcbnn_amd.device import DeviceView
    E = _lib().TcbnnError

    def view(rows, cols, wide):
        v = DeviceView.of(torch.zeros((rows, wide))[:, :cols])
        return DeviceView(P, v.nbytes, v.ld, shape=v.shape)

    buf, raw = DeviceView(P, 4096), DeviceView(P, 4 * (7 * 12 + 8), 12)  # (raw: eight rows of eight, twelve apart, and no byte more)
    linear = lambda x, w=buf, b=None, y=buf: head.LinearLayerParam("l", 8, 8, 8).initialize(w, b, x, output_gpu=y)  # noqa: E731
    assert view(8, 8, 12).shape == (8, 8) and raw.shape is None
    for good in (view(8, 8, 12), view(9, 9, 12), view(8, 8, 8), view(1, 64, 64), raw):
        linear(good)
        linear(buf, w=good, y=good)
    with pytest.raises(E, match="input.*rows"):
        linear(view(2, 32, 40))  # 64 values, but eight rows of 40 would go past them
    with pytest.raises(E, match="input.*rows"):
        linear(view(4, 16, 16))
    with pytest.raises(E, match="input.*rows"):
        linear(view(16, 4, 12))  # eight values of its rows are there, four of them in the gap
    with pytest.raises(E, match="weight.*rows"):
        linear(buf, w=DeviceView(P, 4 * (7 * 12 + 7), 12))
    with pytest.raises(E, match="output.*rows"):
        linear(buf, y=view(4, 16, 24))
    with pytest.raises(E, match="bias.*gaps"):
        linear(buf, b=view(8, 1, 12))  # a column
    linear(buf, b=view(8, 1, 1))
    linear(buf, b=view(2, 4, 4))
    with pytest.raises(E, match="gamma.*gaps"):
        head.LayerNormLayerParam("n", 4, 8).initialize(DeviceView(P, 64, 2), None, buf, output_gpu=buf, mean_gpu=buf, rstd_gpu=buf)
    outs = dict(logprob_gpu=buf, entropy_gpu=buf, logsumexp_gpu=buf, rank_gpu=buf)
    best = head.LogProbsLayerParam("p", 8, 64, top=4)
    best.initialize(buf, buf, **outs, top_index_gpu=view(8, 4, 4), top_logprob_gpu=view(1, 32, 32))
    with pytest.raises(E, match="top_index.*gaps"):
        best.initialize(buf, buf, **outs, top_index_gpu=view(8, 4, 6), top_logprob_gpu=buf)


def test_downloads_refuse_gaps():
    """download_output() copies one piece of memory: not where its rows have others between them."""
    from tcbnn_amd import head
    from tcbnn_amd.device import DeviceView
    copied = []

    class View(DeviceView):
        def to_numpy(self, dtype, shape):
            copied.append(shape)
            return np.zeros(shape, dtype)

    buf = View(P, 4096)
    linear = lambda y: head.LinearLayerParam("l", 8, 8, 8).initialize(buf, None, buf, output_gpu=y)  # noqa: E731
    norm = lambda y: head.LayerNormLayerParam("n", 8, 8).initialize(None, None, buf, output_gpu=y, mean_gpu=buf, rstd_gpu=buf)  # noqa: E731
    for layer in (linear, norm):
        with pytest.raises(_lib().TcbnnError, match="gaps"):
            layer(View(P, 4096, 12)).download_output()
        assert not copied
        for y in (buf, View(P, 4096, 8)):
            assert layer(y).download_output().shape == (8, 8) and copied.pop() == (8, 8)
    one = head.LinearLayerParam("l", 1, 8, 8).initialize(buf, None, buf, output_gpu=View(P, 4096, 12))  # (one row has none)
    assert one.download_output().shape == (1, 8)


def test_layers_are_initialized_anew():
    """initialize() once more: no call of the layer still uses the buffers of before, and it keeps none of its own from there."""
    from tcbnn_amd import head
    from tcbnn_amd.device import DeviceView
    E, alive = _lib().TcbnnError, []

    class Own(DeviceView):
        def __init__(self, nbytes):
            super().__init__(P, nbytes)
            alive.append(self)

    def fill(layer):
        layer._buffer = lambda nbytes: layer._owned.append(Own(nbytes)) or layer._owned[-1]
        return layer

    def started(layer):
        args = {"l": (buf, None, buf), "n": (None, None, buf), "p": (buf, buf)}[layer.name]
        return layer.initialize(*args)

    buf, short = DeviceView(P, 4096), DeviceView(P, 16)
    layers = [fill(head.LinearLayerParam("l", 8, 8, 8)), fill(head.LayerNormLayerParam("n", 8, 8)), fill(head.LogProbsLayerParam("p", 8, 8))]
    grads = {"l": (buf, buf, buf, buf), "n": (buf, buf, buf, buf), "p": (buf, buf, buf)}
    for layer in layers:
        for _ in range(2):
            started(layer)
            with pytest.raises(E, match="not initialized"):
                layer.backward()
            own = len(alive)
            layer.initialize_backward(*grads[layer.name])
            layer.initialize_backward(*grads[layer.name])
            assert {id(b) for b in layer._owned} <= {id(b) for b in alive} and len(layer._owned) <= own + 1
            first = list(alive)
            alive.clear()
            started(layer)
            assert not {id(b) for b in layer._owned} & {id(b) for b in first}
            alive.clear()
        bad = {"l": (buf, None, short), "n": (None, None, short), "p": (short, buf)}[layer.name]
        started(layer).initialize_backward(*grads[layer.name])
        with pytest.raises(E, match="holds"):
            layer.initialize(*bad)
        for call in (layer.forward, layer.backward):
            with pytest.raises(E, match="not initialized"):
                call()


@pytest.mark.parametrize("count", [7, 9, 16])
def test_head_refuses_other_than_a_target_a_row(count):
    """More targets than rows would be counted in the mean of the rows' cross entropy."""
    from tcbnn_amd import head
    from tcbnn_amd.device import DeviceView
    with pytest.raises(_lib().TcbnnError, match="targets"):
        head.FloatHead(8, 16, 16, 4).initialize(DeviceView(P, 4 * 8 * 16), np.zeros(count, np.int32))


def test_encode_rounds_to_nearest_even():
    from tcbnn_amd import head
    torch = pytest.importorskip("torch")
    r = np.random.default_rng(3)
    x = np.concatenate([r.integers(0, 2 ** 32, 20000, dtype=np.uint64).astype(np.uint32).view(np.float32),
                        np.array([0.0, -0.0, np.inf, -np.inf, 1.00390625, 1.01171875, 3.4e38], np.float32)])
    for dtype, t in (("bf16", torch.bfloat16), ("f16", torch.float16), ("f32", torch.float32)):
        want = torch.from_numpy(x).to(t).float().numpy()
        with np.errstate(over="ignore", invalid="ignore"):
            np.testing.assert_array_equal(head.decode(head.encode(x, dtype), dtype), want)


def _differences(f, x, v):
    h = 1e-5
    return (f(x + h * v) - f(x - h * v)) / (2 * h)


@pytest.mark.parametrize("name", ["none", "relu", "gelu", "silu"])
def test_slopes_of_activations(name):
    z = np.linspace(-6, 6, 241) + 0.01234
    np.testing.assert_allclose(_differences(lambda a: ho.act(name, a), z, 1.0), ho.slope(name, z), atol=1e-8)


def test_gradient_formulas_of_norm_and_log_probabilities():
    r = np.random.default_rng(9)
    m, n = 5, 12
    x, gamma, dy, v = (r.standard_normal(s) for s in ((m, n), (n,), (m, n), (m, n)))
    _, mean, rstd = ho.norm(x, gamma, 0.0, 1e-5)
    xh, g = (x - mean[:, None]) * rstd[:, None], dy * gamma
    dx = (g - g.mean(1, keepdims=True) - xh * (g * xh).mean(1, keepdims=True)) * rstd[:, None]
    assert abs(_differences(lambda a: (dy * ho.norm(a, gamma, 0.0, 1e-5)[0]).sum(), x, v) - (dx * v).sum()) < 1e-7
    t, c, ce = 3, 0.7, -0.4
    logprob, entropy, lse, *_ = ho.logprobs(x[0], t, 0)
    p = np.exp(x[0] - lse)
    dx = c * ((np.arange(n) == t) - p) - ce * p * (x[0] - lse + entropy)

    def f(a):
        lp, h, *_ = ho.logprobs(a, t, 0)
        return c * lp + ce * h

    assert abs(_differences(f, x[0], v[0]) - (dx * v[0]).sum()) < 1e-8
