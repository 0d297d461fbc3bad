"""The float head as it is used: on the frozen binary layers of the MLP, trained and scored (the example's command); its passes on
another stream and in a captured graph; calls that allocate nothing."""
import ctypes as C

import numpy as np
import pytest

from tests import headops as ho

pytestmark = pytest.mark.gpu


def _forward(p, x, t):
    """The head's definition in 64 bits: logits, mean cross entropy."""
    n1, _, _ = ho.norm(x, p["gamma1"], p["beta1"], 1e-5)
    h = ho.act("gelu", n1 @ p["w1"].T + p["b1"])
    if h.shape == x.shape:
        h = h + x
    n2, _, _ = ho.norm(h, p["gamma2"], p["beta2"], 1e-5)
    z = n2 @ p["w2"].T + p["b2"]
    given = t >= 0
    lp = z - z.max(1, keepdims=True)
    lp = lp - np.log(np.exp(lp).sum(1, keepdims=True))
    return z, -lp[given, t[given]].sum() / max(1, given.sum())


@pytest.mark.parametrize("rows,hidden,classes", [(50, 256, 10), (33, 96, 17)])
def test_head_on_binary_layers(gpu, rows, hidden, classes):
    """Logits and loss against the definition, parameters' gradients against its central differences."""
    from tcbnn_amd.head import FloatHead
    from tcbnn_amd.head_example import binary_features
    features, _, trunk = binary_features(rows, 256)
    x = features.to_numpy(np.float32, (rows, 256)).astype(np.float64)
    assert set(np.unique(x)) == {-1.0, 1.0}
    r = np.random.default_rng(3)
    t = r.integers(-1, classes, rows).astype(np.int32)
    head = FloatHead(rows, 256, hidden, classes).initialize(features, t, seed=4)
    head.forward()
    head.backward()
    p = {k: v.astype(np.float64) for k, v in head.params.items()}
    z, loss = _forward(p, x, t)
    # about a thousand fp32 roundings between the features and a logit, of values of a few units
    np.testing.assert_allclose(head.linear2.download_output(), z, atol=1000 * ho.U32 * np.abs(z).max())
    assert abs(head.loss() - loss) < 1e-5
    for name, g in head.gradients().items():
        v = r.standard_normal(p[name].shape)
        d = [_forward({**p, name: p[name] + s * 1e-5 * v}, x, t)[1] for s in (1, -1)]
        assert abs((g * v).sum() - (d[0] - d[1]) / 2e-5) <= 1000 * ho.U32 * np.abs(g * v).sum() + 1e-6, name
    head.release()
    trunk.release()


@pytest.mark.parametrize("dtype", ho.DTYPES)
def test_example_learns(gpu, capsys, dtype):
    from tcbnn_amd import head_example
    losses = head_example.main(["--batch", "512", "--hidden", "256", "--steps", "12", "--rate", "0.1", "--dtype", dtype])
    assert losses[-1] < 0.85 * losses[0]  # (in 64 bits: 2.696 to 2.131)
    assert "best classes" in capsys.readouterr().out


def test_passes_on_a_stream_and_in_a_graph(gpu):
    """Forward and backward captured into a graph and replayed: the same bits as the eager passes, every time, with eager work
    between the replays; rows and sizes that take several kernels each."""
    from tcbnn_amd import _lib
    from tcbnn_amd.device import Graph, Stream
    from tcbnn_amd.head import FloatHead
    r = np.random.default_rng(8)
    rows, k, h, c = 300, 264, 500, 20000
    x = ho.Matrix(r.standard_normal((rows, k)), "bf16")
    t = r.integers(0, c, rows).astype(np.int32)
    head = FloatHead(rows, k, h, c, "bf16", top=7).initialize(x.view, t)
    stream = Stream()

    def passes(s):
        head.forward(s)
        head.backward(s)

    def results():
        out = head.logprobs.download_output()
        return {**out, **head.gradients()}

    passes(stream)
    stream.synchronize()
    want = results()
    graph = Graph(stream, passes)
    for _ in range(4):
        for buf in head._flows + list(head._grads.values()):
            buf.fill(0xA5)
        head.logprobs.logprob_gpu.fill(0xA5)
        _lib.device_synchronize()
        graph.launch()
        stream.synchronize()
        for name, a in results().items():
            np.testing.assert_array_equal(a, want[name], err_msg=name)
        passes(None)
        _lib.device_synchronize()
        for name, a in results().items():
            np.testing.assert_array_equal(a, want[name], err_msg=name)
    head.release()


def test_calls_allocate_nothing(gpu):
    from tcbnn_amd import _lib
    from tcbnn_amd.head import FloatHead
    r = np.random.default_rng(9)
    x = ho.Matrix(r.standard_normal((70, 1000)), "f16")
    head = FloatHead(70, 1000, 1000, 40000, "f16").initialize(x.view, r.integers(0, 40000, 70).astype(np.int32))
    free, total = C.c_size_t(0), C.c_size_t(0)
    head.forward()
    head.backward()
    _lib.device_synchronize()
    _lib.hip.hipMemGetInfo(C.byref(free), C.byref(total))
    before = free.value
    for _ in range(3):
        head.forward()
        head.backward()
    _lib.device_synchronize()
    _lib.hip.hipMemGetInfo(C.byref(free), C.byref(total))
    assert free.value == before
    head.release()
