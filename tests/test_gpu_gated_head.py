"""The gated block's operators together, as they are used: a head of gated residual blocks on the frozen binary layers of the MLP, trained
and scored (the example's command); its passes on another stream and in captured graphs; calls that allocate nothing."""
import ctypes as C

import numpy as np
import pytest

from tests import blockops as bo
from tests import headops as ho

pytestmark = pytest.mark.gpu

SCALE = 0.5


def _forward(p, x, t, blocks):
    """The head's definition in 64 bits: what the loss reads, the rows' losses, their mean."""
    def rms(v):
        return v / np.sqrt((v * v).mean(1, keepdims=True) + np.float64(np.float32(1e-5)))

    stream, y = x, rms(x) * p["gamma"]
    for i in range(blocks):
        z = y @ p["w_gated%d" % i].T + p["b_gated%d" % i]
        n = z.shape[1] // 2
        block = (ho.act("silu", z[:, :n]) * z[:, n:]) @ p["w_down%d" % i].T
        stream = stream + SCALE * p["gate%d" % i] * rms(block) * p["gamma_after%d" % i]
        y = rms(stream) * p["gamma_before%d" % i]
    loss = bo.loss(y, p["w_class"], p["b_class"], t)[0]
    return y, loss, loss.sum() / max(1, (t >= 0).sum())


@pytest.mark.parametrize("rows,hidden,classes,blocks", [(50, 256, 10, 1), (33, 96, 300, 2), (300, 40, 33, 3)])
def test_head_on_binary_layers(gpu, rows, hidden, classes, blocks):
    """Losses against the definition, parameters' gradients against its central differences."""
    from tcbnn_amd.head import GatedHead
    from tcbnn_amd.head_example import binary_features
    features, _, trunk = binary_features(rows, 256)
    x = features.to_numpy(np.float32, (rows, 256)).astype(np.float64)
    r = np.random.default_rng(3)
    t = r.integers(-1, classes, rows).astype(np.int32)
    head = GatedHead(rows, 256, hidden, classes, blocks=blocks, scale=SCALE).initialize(features, t, seed=4)
    for name, a in head.params.items():  # (nothing at its first value)
        a += 0.1 * r.standard_normal(a.shape).astype(np.float32)
        head._devices[name].upload(a)
    head.forward()
    head.backward()
    p = {k: v.astype(np.float64) for k, v in head.params.items()}
    y, losses, mean = _forward(p, x, t, blocks)
    # about a thousand fp32 roundings a block between the features and a logit, of values of a few units
    np.testing.assert_allclose(head.linear_loss.download_output()["loss"], losses, atol=1000 * blocks * ho.U32 * 30)
    assert abs(head.loss() - mean) < 1e-4
    for name, g in head.gradients().items():
        v = r.standard_normal(p[name].shape)
        d = [_forward({**p, name: p[name] + s * 1e-5 * v}, x, t, blocks)[2] for s in (1, -1)]
        assert abs((g * v).sum() - (d[0] - d[1]) / 2e-5) <= 3000 * blocks * ho.U32 * np.abs(g * v).sum() + 1e-6, name
    scores = head.score()
    np.testing.assert_allclose(scores["logprob"], -losses, atol=1000 * blocks * ho.U32 * 30)
    np.testing.assert_array_equal(scores["rank"] < 0, t < 0)
    head.release()
    trunk.release()


@pytest.mark.parametrize("dtype", ho.DTYPES)
def test_example_runs(gpu, capsys, dtype):
    from tcbnn_amd import head_example
    losses = head_example.main(["--batch", "256", "--hidden", "256", "--steps", "2", "--rate", "0.1", "--dtype", dtype, "--head", "gated", "--blocks", "2"])
    assert len(losses) == 3 and np.isfinite(losses).all()
    assert "best classes" in capsys.readouterr().out


def _head(rows, k, h, c, dtype, blocks, seed):
    from tcbnn_amd.head import GatedHead
    r = np.random.default_rng(seed)
    x = ho.Matrix(r.standard_normal((rows, k)), dtype)
    return GatedHead(rows, k, h, c, dtype, blocks=blocks).initialize(x.view, r.integers(-1, c, rows).astype(np.int32)), x


def _results(head):
    return {**head.linear_loss.download_output(), **head.gradients()}


@pytest.mark.parametrize("rows,k,h,c,dtype", [(300, 264, 500, 20000, "bf16"), (20, 72, 40, 33, "f16"), (2100, 256, 256, 1030, "bf16"), (40, 61, 77, 90, "f32")])
def test_passes_on_streams_and_in_graphs(gpu, rows, k, h, c, dtype):
    """Forward and backward captured into a graph and replayed: the same bits as the eager passes, every time, with eager work between the replays;
    two heads with graphs of their own, replayed in turn on streams of their own."""
    from tcbnn_amd import _lib
    from tcbnn_amd.device import Graph, Stream
    pairs = [_head(rows, k, h, c, dtype, 2, seed) for seed in (8, 9)]
    heads, streams, graphs, wants = [p[0] for p in pairs], [Stream(), Stream()], [], []

    def passes(head):
        def go(s):
            head.forward(s)
            head.backward(s)
        return go

    for head, stream in zip(heads, streams):
        passes(head)(stream)
        stream.synchronize()
        wants.append(_results(head))
        graphs.append(Graph(stream, passes(head)))
    for _ in range(3):
        for head in heads:
            for buf in head._flows + list(head._grads.values()):
                buf.fill(0xA5)
        _lib.device_synchronize()
        for g in graphs:
            g.launch()
        for s in streams:
            s.synchronize()
        for head, want in zip(heads, wants):
            for name, a in _results(head).items():
                np.testing.assert_array_equal(a, want[name], err_msg=name)
        for head in heads:
            passes(head)(None)
        _lib.device_synchronize()
        for head, want in zip(heads, wants):
            for name, a in _results(head).items():
                np.testing.assert_array_equal(a, want[name], err_msg=name)
    for head in heads:
        head.release()


def test_sums_in_one_order(gpu):
    """The same bits in every call, whatever was in the workspaces: sizes that take splits, pieces, planes and joins."""
    from tcbnn_amd import _lib, head as hd
    r = np.random.default_rng(12)
    for m, k, n, dtype in ((64, 4096, 600, "bf16"), (333, 200, 3003, "f16"), (70000, 24, 2100, "bf16")):
        x, w = ho.Matrix(r.standard_normal((m, k)), dtype, shift=0), ho.Matrix(r.standard_normal((n, k)) / 8, dtype, shift=0)
        dx, dw, db = ho.Matrix(None, dtype, 0, m, k), ho.Matrix(None, dtype, 0, n, k), ho.empty(n)
        layer = hd.LinearLossLayerParam("loss", m, k, n, dtype).initialize(w.view, None, x.view, ho.vector(r.integers(0, n, m), np.int32))
        layer.initialize_backward(ho.vector(np.ones(m)), dx.view, dw.view, db)
        first = None
        for fill in (0, 0xFF, 0x3C):
            for buf in layer._owned:
                if buf not in (layer.loss_gpu, layer.logsumexp_gpu):
                    buf.fill(fill)
            layer.forward()
            layer.backward()
            _lib.device_synchronize()
            got = [layer.download_output()["loss"], dx.get(), dw.get(), db.to_numpy(np.float32, (n,))]
            first = first or got
            for a, b in zip(got, first):
                np.testing.assert_array_equal(a, b)
        layer.release()


def test_calls_allocate_nothing(gpu):
    from tcbnn_amd import _lib
    head, x = _head(70, 1000, 500, 40000, "f16", 1, 9)
    free, total = C.c_size_t(0), C.c_size_t(0)
    head.forward()
    head.backward()
    head.score()
    _lib.hip.hipMemGetInfo(C.byref(free), C.byref(total))
    before = free.value
    for _ in range(3):
        head.forward()
        head.backward()
        head.score()
    _lib.hip.hipMemGetInfo(C.byref(free), C.byref(total))
    assert free.value == before
    head.release()
