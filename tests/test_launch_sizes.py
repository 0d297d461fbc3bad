"""The float head's launches at the largest sizes that its entry points take, without a GPU: a launch's threads are counted in 32 bits.  Each test runs in a
process of its own with tests/native/launch_stub.c preloaded, so that no kernel is run and no pointer followed."""
import os
import subprocess
import sys
import textwrap

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

PRELUDE = """
import ctypes as C
from tcbnn_amd import _lib
L, stub = _lib.lib, C.CDLL(STUB)
P, DTYPES, LARGE = 1 << 20, _lib.DTYPES, 1 << 62
def launches(entry, desc):
    n = C.c_int.in_dll(stub, "stub_launches")
    n.value = 0
    assert getattr(L, entry)(C.byref(desc), None) == 0, L.tcbnn_last_error()
    assert 0 < n.value <= 4096
    grids, groups = ((C.c_uint * 4096).in_dll(stub, "stub_" + name)[:n.value] for name in ("grids", "groups"))
    for grid, group in zip(grids, groups):
        assert 0 < grid * group < 1 << 32, (entry, grid, group)
    return list(zip(grids, groups))
"""


@pytest.fixture(scope="module")
def run(tmp_path_factory):
    so = str(tmp_path_factory.mktemp("native") / "launch_stub.so")
    subprocess.run(["gcc", "-O1", "-shared", "-fPIC", "-o", so, os.path.join(ROOT, "tests/native/launch_stub.c")], check=True)
    preload = ":".join([so] + [v for v in [os.environ.get("LD_PRELOAD")] if v])
    env = dict(os.environ, LD_PRELOAD=preload, PYTHONPATH=ROOT, OMP_NUM_THREADS="1", OPENBLAS_NUM_THREADS="1")

    def go(body):
        code = "STUB = %r\n" % so + PRELUDE + textwrap.dedent(body) + "\nprint('done')\n"
        p = subprocess.run([sys.executable, "-c", code], env=env, stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True, timeout=240)
        assert p.returncode == 0 and p.stdout.strip().endswith("done"), "exit %d: %s" % (p.returncode, p.stdout[-2000:])
    return go


def test_launches_are_seen(run):
    run("""
    d = _lib.LinearDesc(input=P, weight=P, output=P, rows=1, in_features=4096, out_features=4096, dtype=DTYPES["bf16"])
    assert launches("tcbnn_linear_forward", d) == [(256, 512)]
    """)


def test_few_rows_of_many_outputs(run):
    """The kernel for few rows has 16 outputs of a workgroup of 512 threads; the loss's gradients of four rows and less always take it."""
    run("""
    inputs, n, dt = 4096, 1 << 28, DTYPES["bf16"]
    def few(entry, desc):
        assert sum(grid for grid, group in launches(entry, desc) if group == 512) == n // 16, entry
    few("tcbnn_linear_forward", _lib.LinearDesc(input=P, weight=P, output=P, rows=1, in_features=inputs, out_features=n, dtype=dt))
    few("tcbnn_gated_forward", _lib.GatedDesc(input=P, weight=P, output=P, rows=1, in_features=inputs, features=n // 2, dtype=dt, activation=3))
    few("tcbnn_linear_loss_forward", _lib.LinearLossDesc(input=P, weight=P, targets=P, loss=P, rows=1, in_features=inputs, classes=n, dtype=dt, workspace=P, workspace_bytes=LARGE))
    for rows in (1, 4):
        few("tcbnn_linear_loss_backward", _lib.LinearLossGradDesc(input=P, weight=P, targets=P, logsumexp=P, loss=P, grad_loss=P, grad_input=P, grad_weight=P, grad_bias=P, rows=rows,
                                                                  in_features=inputs, classes=n, dtype=dt, workspace=P, workspace_bytes=LARGE))
    """)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
def test_the_largest_sizes(run, dtype):
    """Rows, inputs and outputs at their limits, the others small."""
    run("""
    dt, many, wide, outs = DTYPES[%r], (1 << 31) - (1 << 22), 1 << 20, 1 << 28
    for m, k, n in ((many, 8, 3), (many, 1, 64), (3, wide, 40), (700, wide, 2000), (7, 16, outs), (16, 1024, outs), (300, 8, outs), (17, 1, outs), (1, 4096, outs)):
        launches("tcbnn_linear_forward", _lib.LinearDesc(input=P, weight=P, output=P, rows=m, in_features=k, out_features=n, dtype=dt))
        launches("tcbnn_linear_backward", _lib.LinearGradDesc(input=P, weight=P, preact=P, grad_output=P, grad_input=P, grad_weight=P, grad_bias=P, rows=m, in_features=k,
                                                              out_features=n, dtype=dt, activation=3, workspace=P, workspace_bytes=LARGE))
        launches("tcbnn_linear_loss_forward", _lib.LinearLossDesc(input=P, weight=P, targets=P, loss=P, rows=m, in_features=k, classes=n, dtype=dt, workspace=P,
                                                                  workspace_bytes=LARGE))
        if m * n < 1 << 33:  # (pieces beyond are more launches than are kept here)
            launches("tcbnn_linear_loss_backward", _lib.LinearLossGradDesc(input=P, weight=P, targets=P, logsumexp=P, loss=P, grad_loss=P, grad_input=P, grad_weight=P,
                                                                           grad_bias=P, rows=m, in_features=k, classes=n, dtype=dt, workspace=P, workspace_bytes=LARGE))
        n = n // 2 + 1 if n < outs else n // 2
        launches("tcbnn_gated_forward", _lib.GatedDesc(input=P, weight=P, output=P, preact=P, rows=m, in_features=k, features=n, dtype=dt, activation=3, workspace=P,
                                                       workspace_bytes=LARGE))
        launches("tcbnn_gated_backward", _lib.GatedGradDesc(input=P, weight=P, preact=P, grad_output=P, grad_input=P, grad_weight=P, grad_bias=P, rows=m, in_features=k,
                                                            features=n, dtype=dt, activation=3, workspace=P, workspace_bytes=LARGE))
    for m, n in (((1 << 31) - 1, 8), ((1 << 31) - 1, 700), (1 << 24, 65536), (1, 65536)):
        for after, before in ((1, 1), (2, 2)):
            launches("tcbnn_blocknorm_forward", _lib.BlockNormDesc(stream_in=P, block=2 * P, stream_out=3 * P, output=4 * P, rows=m, features=n, dtype=dt, after=after, before=before,
                                                                   scale=1.0, eps=1e-5))
            launches("tcbnn_blocknorm_backward", _lib.BlockNormGradDesc(stream_out=P, block=P, after_rstd=P, after_mean=P, before_rstd=P, before_mean=P, grad_output=P,
                                                                        grad_stream_out=P, grad_stream_in=2 * P, grad_block=3 * P, grad_gate=P, rows=m, features=n, dtype=dt,
                                                                        after=after, before=before, scale=1.0, workspace=P, workspace_bytes=LARGE))
    """ % dtype)
