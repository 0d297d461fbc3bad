"""The gated block's operators without a GPU: what their entry points refuse (nothing is launched), what their layers refuse, and the
definitions that the GPU tests compare with, against differences."""
import ctypes as C

import numpy as np
import pytest

from tests import blockops as bo

EINVAL, ENULL = -1, -2
P = 0x1000  # a pointer that no refused call follows


def _lib():
    from tcbnn_amd import _lib
    return _lib


def _norms(**kw):
    d = dict(stream_in=P, block=P + 64, stream_out=P + 128, output=P + 256, rows=4, features=8, dtype=1, after=2, before=1, scale=1.0, eps=1e-5)
    return "tcbnn_blocknorm_forward", _lib().BlockNormDesc(**{**d, **kw})


def _norms_grad(**kw):
    d = dict(stream_out=P, block=P + 64, after_rstd=P, after_mean=P, before_rstd=P, before_mean=P, grad_output=P + 128, grad_stream_out=P + 256,
             grad_stream_in=P + 512, grad_block=P + 1024, grad_gate=P, rows=4, features=8, dtype=1, after=2, before=1, scale=1.0, workspace=P,
             workspace_bytes=1 << 30)
    return "tcbnn_blocknorm_backward", _lib().BlockNormGradDesc(**{**d, **kw})


def _gated(**kw):
    d = dict(input=P, weight=P, output=P, rows=4, in_features=8, features=8, dtype=1, activation=3)
    return "tcbnn_gated_forward", _lib().GatedDesc(**{**d, **kw})


def _gated_grad(**kw):
    d = dict(input=P, weight=P, preact=P, grad_output=P, grad_input=P, grad_weight=P, grad_bias=P, rows=4, in_features=8, features=8, dtype=1,
             activation=3, workspace=P, workspace_bytes=1 << 30)
    return "tcbnn_gated_backward", _lib().GatedGradDesc(**{**d, **kw})


def _loss(**kw):
    d = dict(input=P, weight=P, targets=P, loss=P, logsumexp=P, rows=4, in_features=8, classes=8, dtype=1, workspace=P, workspace_bytes=1 << 30)
    return "tcbnn_linear_loss_forward", _lib().LinearLossDesc(**{**d, **kw})


def _loss_grad(**kw):
    d = dict(input=P, weight=P, targets=P, logsumexp=P, grad_loss=P, grad_input=P, grad_weight=P, grad_bias=P, rows=4, in_features=8, classes=8, dtype=1,
             workspace=P, workspace_bytes=1 << 30)
    return "tcbnn_linear_loss_backward", _lib().LinearLossGradDesc(**{**d, **kw})


@pytest.mark.parametrize("make,change,code,message", [
    (_loss, dict(dtype=3), EINVAL, "dtype"), (_loss, dict(rows=-1), EINVAL, "shape"), (_loss, dict(in_features=0), EINVAL, "shape"),
    (_loss, dict(classes=0), EINVAL, "shape"), (_loss, dict(in_features=(1 << 20) + 1), EINVAL, "inputs"), (_loss, dict(classes=(1 << 28) + 1), EINVAL, "classes"),
    (_loss, dict(rows=(1 << 31) - 1), EINVAL, "rows"), (_loss, dict(input_ld=7), EINVAL, "overlap"), (_loss, dict(weight_ld=-8), EINVAL, "overlap"),
    (_loss, dict(weight_ld=1 << 23), EINVAL, "apart"), (_loss, dict(input_ld=1 << 40), EINVAL, "apart"), (_loss, dict(input=0), ENULL, "input"),
    (_loss, dict(weight=0), ENULL, "weight"), (_loss, dict(targets=0), ENULL, "targets"), (_loss, dict(workspace=0), ENULL, "workspace"),
    (_loss, dict(workspace=P + 8), EINVAL, "aligned"), (_loss, dict(workspace_bytes=16), EINVAL, "workspace"),
    (_loss_grad, dict(dtype=-1), EINVAL, "dtype"), (_loss_grad, dict(rows=-3), EINVAL, "shape"), (_loss_grad, dict(grad_input_ld=4), EINVAL, "overlap"),
    (_loss_grad, dict(grad_weight_ld=4), EINVAL, "overlap"), (_loss_grad, dict(weight_ld=1 << 23), EINVAL, "apart"), (_loss_grad, dict(input=0), ENULL, "input"),
    (_loss_grad, dict(weight=0), ENULL, "weight"), (_loss_grad, dict(targets=0), ENULL, "targets"), (_loss_grad, dict(logsumexp=0), ENULL, "logsumexp"),
    (_loss_grad, dict(grad_loss=0), ENULL, "grad_loss"), (_loss_grad, dict(workspace=0), ENULL, "workspace"),
    (_loss_grad, dict(workspace=P + 4), EINVAL, "aligned"), (_loss_grad, dict(workspace_bytes=64), EINVAL, "workspace"),
    (_gated, dict(dtype=3), EINVAL, "dtype"), (_gated, dict(activation=4), EINVAL, "activation"), (_gated, dict(rows=-1), EINVAL, "shape"),
    (_gated, dict(in_features=0), EINVAL, "shape"), (_gated, dict(features=0), EINVAL, "shape"), (_gated, dict(in_features=(1 << 20) + 1), EINVAL, "inputs"),
    (_gated, dict(features=(1 << 27) + 1), EINVAL, "features"), (_gated, dict(rows=(1 << 31) - 1), EINVAL, "rows"),
    (_gated, dict(input_ld=7), EINVAL, "overlap"), (_gated, dict(weight_ld=7), EINVAL, "overlap"), (_gated, dict(output_ld=7), EINVAL, "overlap"),
    (_gated, dict(preact_ld=15), EINVAL, "overlap"), (_gated, dict(input=0), ENULL, "input"), (_gated, dict(weight=0), ENULL, "weight"),
    (_gated, dict(output=0), ENULL, "output"),
    (_gated_grad, dict(dtype=9), EINVAL, "dtype"), (_gated_grad, dict(activation=-1), EINVAL, "activation"), (_gated_grad, dict(rows=-4), EINVAL, "shape"),
    (_gated_grad, dict(grad_output=0), ENULL, "grad_output"), (_gated_grad, dict(preact=0), ENULL, "preact"), (_gated_grad, dict(input=0), ENULL, "input"),
    (_gated_grad, dict(weight=0), ENULL, "weight"), (_gated_grad, dict(workspace=0), ENULL, "workspace"), (_gated_grad, dict(workspace=P + 4), EINVAL, "aligned"),
    (_gated_grad, dict(workspace_bytes=1), EINVAL, "workspace"), (_gated_grad, dict(grad_weight_ld=4), EINVAL, "overlap"),
    (_gated_grad, dict(preact_ld=15), EINVAL, "overlap"), (_gated_grad, dict(features=(1 << 27) + 1), EINVAL, "features"),
    (_norms, dict(dtype=3), EINVAL, "dtype"), (_norms, dict(after=3), EINVAL, "norm"), (_norms, dict(before=-1), EINVAL, "norm"),
    (_norms, dict(rows=-1), EINVAL, "shape"), (_norms, dict(features=0), EINVAL, "shape"), (_norms, dict(features=65537), EINVAL, "features"),
    (_norms, dict(scale=float("inf")), EINVAL, "scale"), (_norms, dict(scale=float("nan")), EINVAL, "scale"),
    (_norms, dict(eps=-1.0), EINVAL, "eps"), (_norms, dict(eps=float("nan")), EINVAL, "eps"),
    (_norms, dict(stream_in_ld=7), EINVAL, "overlap"), (_norms, dict(block_ld=7), EINVAL, "overlap"),
    (_norms, dict(stream_out_ld=-8), EINVAL, "overlap"), (_norms, dict(output_ld=1), EINVAL, "overlap"),
    (_norms, dict(stream_in=0), ENULL, "stream_in"), (_norms, dict(output=0), ENULL, "output"),
    (_norms, dict(block=0), EINVAL, "block"), (_norms, dict(block=0, after=0, gate=P), EINVAL, "block"),
    (_norms, dict(before=0), EINVAL, "output"), (_norms, dict(before=0, output=0, stream_out=0), EINVAL, "nothing"),
    (_norms, dict(stream_out=P + 256), EINVAL, "one buffer"), (_norms, dict(stream_out=P, stream_out_ld=16), EINVAL, "stride"),
    (_norms, dict(output=P + 64, output_ld=16), EINVAL, "stride"), (_norms, dict(after=1, after_beta=P), EINVAL, "after_beta"),
    (_norms, dict(before_beta=P), EINVAL, "before_beta"), (_norms, dict(after=0, after_gamma=P), EINVAL, "after_gamma"),
    (_norms, dict(before=0, output=0, before_gamma=P), EINVAL, "before_gamma"),
    (_norms_grad, dict(dtype=-1), EINVAL, "dtype"), (_norms_grad, dict(after=9), EINVAL, "norm"), (_norms_grad, dict(rows=-2), EINVAL, "shape"),
    (_norms_grad, dict(features=1 << 17), EINVAL, "features"), (_norms_grad, dict(scale=float("nan")), EINVAL, "scale"),
    (_norms_grad, dict(stream_out=0), ENULL, "stream_out"), (_norms_grad, dict(block=0), ENULL, "block"),
    (_norms_grad, dict(block=0, grad_block=0), ENULL, "block"), (_norms_grad, dict(after_rstd=0), ENULL, "after_rstd"),
    (_norms_grad, dict(after_mean=0), ENULL, "after_mean"), (_norms_grad, dict(before_rstd=0), ENULL, "before_rstd"),
    (_norms_grad, dict(before=2, before_mean=0), ENULL, "before_mean"), (_norms_grad, dict(before=0), EINVAL, "grad"),
    (_norms_grad, dict(grad_block=P + 512), EINVAL, "one buffer"), (_norms_grad, dict(grad_stream_in_ld=3), EINVAL, "overlap"),
    (_norms_grad, dict(grad_stream_in=P + 128, grad_stream_in_ld=16), EINVAL, "stride"),
    (_norms_grad, dict(grad_block=P + 64, grad_block_ld=9), EINVAL, "stride"), (_norms_grad, dict(workspace=0), ENULL, "workspace"),
    (_norms_grad, dict(workspace_bytes=8), EINVAL, "workspace"), (_norms_grad, dict(workspace=P + 2), EINVAL, "aligned"),
    (_norms_grad, dict(grad_before_beta=P), EINVAL, "grad_before_beta"), (_norms_grad, dict(after=1, grad_after_beta=P), EINVAL, "grad_after_beta"),
    (_norms_grad, dict(after=0, grad_after_gamma=P), EINVAL, "grad_after_gamma"), (_norms_grad, dict(after=1, after_beta=P), EINVAL, "after_beta"),
    (_norms_grad, dict(before=0, grad_output=0, grad_before_gamma=P), EINVAL, "grad_before_gamma"),
])
def test_refusals(make, change, code, message):
    entry, d = make(**change)
    lib = _lib().lib
    assert getattr(lib, entry)(C.byref(d), None) == code
    assert message in lib.tcbnn_last_error().decode()


def test_no_rows_and_null_descriptors():
    lib = _lib().lib
    for entry, d in (_norms(rows=0, stream_in=0, output=0), _gated(rows=0, input=0, output=0),
                     _loss(rows=0, input=0, workspace=0), _loss(loss=0, logsumexp=0, input=0, workspace=0)):
        assert getattr(lib, entry)(C.byref(d), None) == 0
    for entry in ("tcbnn_blocknorm_forward", "tcbnn_blocknorm_backward", "tcbnn_gated_forward", "tcbnn_gated_backward",
                  "tcbnn_linear_loss_forward", "tcbnn_linear_loss_backward"):
        assert getattr(lib, entry)(None, None) == ENULL


def test_workspaces_of_refused_sizes_are_empty():
    lib = _lib().lib
    assert lib.tcbnn_blocknorm_grad_workspace_bytes(0, 8, 0) == lib.tcbnn_blocknorm_grad_workspace_bytes(4, 65537, 0) == 0
    assert lib.tcbnn_blocknorm_grad_workspace_bytes(4, 8, 5) == 0
    assert lib.tcbnn_gated_workspace_bytes(0, 8, 8, 0) == lib.tcbnn_gated_workspace_bytes(4, 8, 0, 0) == lib.tcbnn_gated_workspace_bytes(4, 8, 8, 5) == 0
    assert lib.tcbnn_gated_grad_workspace_bytes(0, 8, 8, 0, 1) == lib.tcbnn_gated_grad_workspace_bytes(4, 8, 0, 0, 0) == 0
    for f in (lib.tcbnn_linear_loss_workspace_bytes, lib.tcbnn_linear_loss_grad_workspace_bytes):
        for a in (0, 1):
            assert f(0, 8, 8, 0, a) == f(4, 0, 8, 0, a) == f(4, 8, -1, 0, a) == f(4, 8, 8, 3, a) == f(4, (1 << 20) + 1, 8, 0, a) == f(4, 8, (1 << 28) + 1, 0, a) == 0
    assert lib.tcbnn_gated_grad_workspace_bytes(4, 8, (1 << 27) + 1, 0, 1) == lib.tcbnn_gated_grad_workspace_bytes(4, 8, 8, 3, 0) == 0


def test_layers_refuse():
    from tcbnn_amd import head
    from tcbnn_amd._lib import TcbnnError
    from tcbnn_amd.device import DeviceView
    with pytest.raises(TcbnnError, match="norm"):
        head.BlockNormLayerParam("norms", 4, 8, "bf16", after="batch")
    with pytest.raises(TcbnnError, match="dtype"):
        head.BlockNormLayerParam("norms", 4, 8, "f64")
    layer = head.BlockNormLayerParam("norms", 4, 8, "bf16", "none", "none")
    x = DeviceView(P, 64)
    with pytest.raises(TcbnnError, match="not initialized"):
        layer.forward()
    with pytest.raises(TcbnnError, match="NULL"):
        layer.initialize(None)
    with pytest.raises(TcbnnError, match="block holds"):
        layer.initialize(x, DeviceView(P, 62))
    with pytest.raises(TcbnnError, match="gate is bf16"):
        layer.initialize(x, x, gate=DeviceView(P, 32, dtype="bf16"), new_stream_gpu=x)
    layer.initialize(x, x, new_stream_gpu=x)
    with pytest.raises(TcbnnError, match="grad_stream"):
        layer.initialize_backward(None, x, DeviceView(P, 8))


def test_gated_kernel_names():
    """The kernel of a forward call by sizes and alignment; nothing is followed."""
    lib = _lib().lib

    def name(**kw):
        d = _gated(**{**dict(rows=64, in_features=1024, features=64), **kw})[1]
        buf = C.create_string_buffer(160)
        assert lib.tcbnn_gated_kernel_name(C.byref(d), buf, 160) == 0
        return buf.value.decode()

    assert name(rows=1) == "gated_few_rows_kernel<__bf16, 8>"
    assert name() == "gated_product_kernel<__bf16, 32, 32, 1, 1, 4, 8, (Access)0, 1, false>"
    assert name(input=P + 2) == "gated_product_kernel<__bf16, 32, 32, 1, 1, 4, 2, (Access)1, 4, true>"
    assert name(in_features=7) == "gated_product_kernel<__bf16, 32, 32, 1, 1, 4, 2, (Access)2, 1, false>"
    assert name(rows=8192, features=4096, dtype=0) == "gated_product_kernel<float, 256, 256, 2, 4, 1, 2, (Access)0, 1, false>"
    d = _gated(rows=-1)[1]
    assert lib.tcbnn_gated_kernel_name(C.byref(d), C.create_string_buffer(8), 8) == EINVAL


def test_gated_layer_refuses():
    from tcbnn_amd import head
    from tcbnn_amd._lib import TcbnnError
    from tcbnn_amd.device import DeviceView
    with pytest.raises(TcbnnError, match="activation"):
        head.GatedLayerParam("gated", 4, 8, 8, "bf16", "tanh")
    layer = head.GatedLayerParam("gated", 4, 8, 8, "bf16")
    x, w = DeviceView(P, 64), DeviceView(P, 256)
    with pytest.raises(TcbnnError, match="weight holds"):
        layer.initialize(DeviceView(P, 255), None, x, output_gpu=x)
    with pytest.raises(TcbnnError, match="preact holds"):
        layer.initialize(w, None, x, output_gpu=x, preact_gpu=x)
    layer.initialize(w, None, x, output_gpu=x)
    with pytest.raises(TcbnnError, match="preact"):
        layer.initialize_backward(x)


def test_loss_layer_refuses():
    from tcbnn_amd import head
    from tcbnn_amd._lib import TcbnnError
    from tcbnn_amd.device import DeviceView
    layer = head.LinearLossLayerParam("loss", 4, 8, 16, "bf16")
    x, w, t = DeviceView(P, 64), DeviceView(P, 256), DeviceView(P, 16)
    with pytest.raises(TcbnnError, match="targets"):
        layer.initialize(w, None, x, None)
    with pytest.raises(TcbnnError, match="targets is i64"):
        layer.initialize(w, None, x, DeviceView(P, 32, dtype="i64"))
    with pytest.raises(TcbnnError, match="weight holds"):
        layer.initialize(x, None, x, t)


def test_copies_are_made_where_they_are_faster():
    """Room for them is asked for by sizes, and only for operands that lie anywhere."""
    lib = _lib().lib
    assert lib.tcbnn_gated_workspace_bytes(64, 1023, 512, 1) == 0  # (a launch more takes longer than it gains)
    assert lib.tcbnn_gated_workspace_bytes(8192, 4095, 4096, 1) >= 2 * 4096 * (8192 + 8192)
    for f in (lib.tcbnn_gated_grad_workspace_bytes, lib.tcbnn_linear_loss_workspace_bytes, lib.tcbnn_linear_loss_grad_workspace_bytes):
        assert f(64, 1023, 512, 1, 0) == f(64, 1023, 512, 1, 1)
        assert f(8192, 4095, 4096, 1, 1) >= f(8192, 4095, 4096, 1, 0) + 2 * 4096 * 8192


def test_loss_keeps_no_logits():
    """Workspaces of a large vocabulary: forward 8 bytes a row and tile, backward a piece of the classes and the sum of the inputs' gradient."""
    lib = _lib().lib
    rows, classes = 8192, 131072
    logits = 2 * rows * classes
    assert lib.tcbnn_linear_loss_workspace_bytes(rows, 1024, classes, 1, 0) < logits / 16
    assert lib.tcbnn_linear_loss_grad_workspace_bytes(rows, 1024, classes, 1, 0) < logits / 4


def test_loss_gradient_is_the_definitions():
    r = np.random.default_rng(6)
    m, k, n = 4, 5, 9
    x, w, b, g = r.standard_normal((m, k)), r.standard_normal((n, k)), r.standard_normal(n), r.standard_normal(m)
    t = np.array([3, -1, 8, 0])

    def total(x, w, b):
        return (g * bo.loss(x, w, b, t)[0]).sum()

    _, _, lse, lse_err, z, zerr, p = bo.loss(x, w, b, t, g)
    got = bo.loss_grads(x, w, t, g, z, zerr, p, lse, lse_err, "f32")
    for name, at in (("input", lambda v: total(x + v, w, b)), ("weight", lambda v: total(x, w + v, b)), ("bias", lambda v: total(x, w, b + v))):
        v = r.standard_normal(got[name][0].shape)
        assert abs((at(1e-5 * v) - at(-1e-5 * v)) / 2e-5 - (got[name][0] * v).sum()) < 1e-7, name


@pytest.mark.parametrize("after", bo.KINDS)
@pytest.mark.parametrize("before", bo.KINDS)
def test_norms_gradient_is_the_definitions(after, before):
    r = np.random.default_rng(5)
    m, n, scale, eps = 3, 7, 0.7, 1e-3
    x, b, dy, ds = (r.standard_normal((m, n)) for _ in range(4))
    p = {k: r.standard_normal(n) for k in ("gate", "ag", "ab", "bg", "bb")}
    if after == "none":
        p["ag"], p["ab"] = np.ones(n), np.zeros(n)
    if before == "none":
        p["bg"], p["bb"] = np.ones(n), np.zeros(n)

    def total(x, b, p):
        s, _, y, _, _, _ = bo.norms(x, b, p["gate"], p["ag"], p["ab"], p["bg"], p["bb"], after, before, scale, eps)
        return (ds * s).sum() + ((dy * y).sum() if before != "none" else 0.0)

    s, _, _, _, first, second = bo.norms(x, b, p["gate"], p["ag"], p["ab"], p["bg"], p["bb"], after, before, scale, eps)
    stats = {"after_mean": first.mean, "after_rstd": first.rstd, "before_mean": second.mean, "before_rstd": second.rstd}
    got = bo.norms_grad(s, b, p["gate"], p["ag"], p["ab"], p["bg"], stats, dy if before != "none" else None, ds, after, before, scale)
    names = {"gate": "gate", "after_gamma": "ag", "after_beta": "ab", "before_gamma": "bg", "before_beta": "bb"}
    for name, (g, _) in got.items():
        if (name.startswith("after") and after == "none") or (name == "after_beta" and after != "layer"):
            continue
        v = r.standard_normal(g.shape)

        def at(t):
            if name == "stream":
                return total(x + t * v, b, p)
            if name == "block":
                return total(x, b + t * v, p)
            return total(x, b, {**p, names[name]: p[names[name]] + t * v})
        h = 1e-5
        assert abs((at(h) - at(-h)) / (2 * h) - (g * v).sum()) < 1e-6, name


def test_gated_head_refuses():
    from tcbnn_amd._lib import TcbnnError
    from tcbnn_amd.device import DeviceView
    from tcbnn_amd.head import GatedHead
    with pytest.raises(TcbnnError, match="blocks"):
        GatedHead(4, 8, 8, 3, blocks=0)
    with pytest.raises(TcbnnError, match="targets"):
        GatedHead(4, 8, 8, 3).initialize(DeviceView(P, 128), np.zeros(3, np.int32))
