"""The floating point end of a network: linear layers, layer norms, log probabilities, gated products, norms around a residual block and
the loss of a linear classifier, forward and backward.

The layers are objects like those of layers.py: a constructor with the sizes, `initialize` with parameters and buffers,
`forward(stream)` and `backward(stream)` as stream-ordered launches that allocate nothing, `download_*` and `release`.
Buffers are DeviceBuffer or DeviceView (memory of another library, with a stride between rows); a parameter may also be
a numpy array, which is uploaded in the layer's type.  What is not given and not asked for is not computed.
All compute goes through the C ABI of libtcbnn_hip.so.  The reference has no counterpart.
"""
import ctypes as C

import numpy as np

from . import _lib
from ._lib import check, lib
from .device import DeviceBuffer


def encode(values, dtype):
    """fp32 values in the bits of `dtype` ("f32", "bf16", "f16"), rounded to nearest even."""
    x = np.ascontiguousarray(values, dtype=np.float32)
    if dtype == "f32":
        return x
    if dtype == "f16":
        return x.astype(np.float16)
    u = x.view(np.uint32).astype(np.uint64)
    bits = ((u + 0x7fff + ((u >> 16) & 1)) >> 16).astype(np.uint16)
    return np.where(np.isnan(x), np.uint16(0x7fc0), bits)


def decode(bits, dtype):
    """What encode() made, as fp32."""
    if dtype == "bf16":
        return (bits.astype(np.uint32) << 16).view(np.float32)
    return bits.astype(np.float32)


def storage(dtype):
    """The numpy type that holds `dtype`."""
    return {"f32": np.float32, "bf16": np.uint16, "f16": np.float16}[dtype]


ITEMSIZE = {"f32": 4, "bf16": 2, "f16": 2, "i32": 4}


def _ptr(buf):
    return None if buf is None else buf.ptr


def _ld(buf):
    return getattr(buf, "ld", 0)


def _anywhere(dtype, cols, *buffers):
    """Whether rows of one of these matrices do not lie at whole 16 bytes."""
    size = ITEMSIZE[dtype]
    return int(any(b.ptr % 16 or (_ld(b) or cols) * size % 16 or cols * size % 16 for b in buffers))


class _HeadLayer:
    def __init__(self, name, dtype):
        if dtype not in _lib.DTYPES:
            raise _lib.TcbnnError("Error: %s: unknown dtype %r" % (name, dtype))
        self.name, self.dtype = name, dtype
        self._forget()

    def _forget(self):
        """As before initialize().  What the layer owned lives on where something else still holds it."""
        self._owned, self._grad_workspace = [], None
        self._desc = self._grad_desc = None  # kept by the calls below
        self._forward = self._backward = self._not_initialized

    def _not_initialized(self, handle):
        raise _lib.TcbnnError("Error: %s: not initialized" % self.name)

    def _buffer(self, nbytes):
        buf = DeviceBuffer(nbytes)
        self._owned.append(buf)
        return buf

    def _grad_buffer(self, nbytes):
        """The backward pass' workspace, in the place of an earlier one."""
        self._backward = self._not_initialized
        self._owned = [buf for buf in self._owned if buf is not self._grad_workspace]
        self._grad_workspace = self._buffer(nbytes) if nbytes else None
        return self._grad_workspace

    def _parameter(self, p, dtype, shape):
        """A parameter's device buffer: what the caller holds, or an upload of a host array."""
        if p is None or hasattr(p, "ptr"):
            return p
        buf = DeviceBuffer.from_numpy(encode(np.asarray(p, np.float32).reshape(shape), dtype))
        self._owned.append(buf)
        return buf

    def _sized(self, buf, what, shape, dtype, gaps=True):
        """`buf`, which holds a matrix or a vector of `shape` in `dtype` (what does not say its type is taken at its size).
        `gaps`: whether rows may be further apart than they are long."""
        if buf is None:
            return buf
        if getattr(buf, "on_host", False):
            raise _lib.TcbnnError("Error: %s: %s lies in host memory" % (self.name, what))
        if getattr(buf, "dtype", None) not in (None, dtype):
            raise _lib.TcbnnError("Error: %s: %s is %s, not %s" % (self.name, what, buf.dtype, dtype))
        rows, cols = shape if len(shape) == 2 else (1, shape[0])
        if buf.nbytes < rows * cols * ITEMSIZE[dtype]:
            raise _lib.TcbnnError("Error: %s: %s holds %d bytes, %d needed" % (self.name, what, buf.nbytes, rows * cols * ITEMSIZE[dtype]))
        ld, there = _ld(buf), getattr(buf, "shape", None)
        if rows * cols == 0:
            pass
        elif ld and (len(shape) == 1 or not gaps):
            if ld != (there[1] if there else cols):
                raise _lib.TcbnnError("Error: %s: %s has gaps between rows" % (self.name, what))
        elif ld and (there[0] < rows or there[1] < cols if there else
                     ((rows - 1) * ld + cols) * ITEMSIZE[dtype] > buf.nbytes):
            raise _lib.TcbnnError("Error: %s: %s is not %d rows of %d, %d apart" % (self.name, what, rows, cols, ld))
        return buf

    def _required(self, buf, what):
        if buf is None:
            raise _lib.TcbnnError("Error: NULL pointer (%s: %s)" % (self.name, what))
        return buf

    def _download(self, buf, rows, cols):
        if rows > 1 and _ld(buf) not in (0, cols):
            raise _lib.TcbnnError("Error: %s: output has gaps between rows" % self.name)
        return decode(buf.to_numpy(storage(self.dtype), (rows, cols)), self.dtype)

    @staticmethod
    def _call(entry, desc):
        """A call of the entry point with this descriptor, on a stream's handle (what does not change is made once: a small
        layer takes no longer on the GPU than its call does here)."""
        ref = C.byref(desc)

        def call(handle):
            rc = entry(ref, handle)
            if rc:
                check(rc)

        return call

    def forward(self, stream=None):
        self._forward(None if stream is None else stream.handle)

    def backward(self, stream=None):
        self._backward(None if stream is None else stream.handle)

    def release(self):
        for buf in self._owned:
            buf.free()
        self._forget()


class LinearLayerParam(_HeadLayer):
    """output = act(input * weight^T + bias) + residual; input [rows][in_features], weight [out_features][in_features]."""

    def __init__(self, name, rows, in_features, out_features, dtype="f32", activation="none"):
        super().__init__(name, dtype)
        if activation not in _lib.ACTIVATIONS:
            raise _lib.TcbnnError("Error: %s: unknown activation %r" % (name, activation))
        self.rows, self.in_features, self.out_features, self.activation = rows, in_features, out_features, activation

    def initialize(self, weight, bias, input_gpu, residual_gpu=None, output_gpu=None, preact_gpu=None, save_preact=False):
        """save_preact: keep the values before the activation, which backward() of a layer with one needs, in a buffer of
        the layer's own (or give `preact_gpu`)."""
        self._forget()
        m, k, n, dt = self.rows, self.in_features, self.out_features, self.dtype
        self.input_gpu = self._sized(self._required(input_gpu, "input"), "input", (m, k), dt)
        self.weight_gpu = self._sized(self._parameter(self._required(weight, "weight"), self.dtype, (n, k)), "weight", (n, k), dt)
        self.bias_gpu = self._sized(self._parameter(bias, "f32", (n,)), "bias", (n,), "f32")
        self.residual_gpu = self._sized(residual_gpu, "residual", (m, n), dt)
        self.output_gpu = self._sized(output_gpu if output_gpu is not None else self._buffer(m * n * ITEMSIZE[dt]), "output", (m, n), dt)
        if preact_gpu is None and save_preact:
            preact_gpu = self._buffer(m * n * ITEMSIZE[dt])
        self.preact_gpu = self._sized(preact_gpu, "preact", (m, n), dt)
        nbytes = lib.tcbnn_linear_workspace_bytes(m, k, n, _lib.DTYPES[self.dtype])
        ws = self._buffer(nbytes) if nbytes else None
        self._desc = _lib.LinearDesc(
            self.input_gpu.ptr, self.weight_gpu.ptr, _ptr(self.bias_gpu), _ptr(self.residual_gpu), self.output_gpu.ptr,
            _ptr(self.preact_gpu), m, k, n, _lib.DTYPES[self.dtype], _lib.ACTIVATIONS[self.activation], _ld(self.input_gpu),
            _ld(self.weight_gpu), _ld(self.residual_gpu), _ld(self.output_gpu), _ld(self.preact_gpu), _ptr(ws), nbytes)
        self._forward = self._call(lib.tcbnn_linear_forward, self._desc)
        return self

    def initialize_backward(self, grad_output_gpu, grad_input_gpu=None, grad_weight_gpu=None, grad_bias_gpu=None):
        """After initialize().  Gradients are written where a buffer is given."""
        m, k, n, dt = self.rows, self.in_features, self.out_features, self.dtype
        if self.activation != "none":
            self._required(self.preact_gpu, "preact")
        self.grad_output_gpu = self._sized(self._required(grad_output_gpu, "grad_output"), "grad_output", (m, n), dt)
        self.grad_input_gpu = self._sized(grad_input_gpu, "grad_input", (m, k), dt)
        self.grad_weight_gpu = self._sized(grad_weight_gpu, "grad_weight", (n, k), dt)
        self.grad_bias_gpu = self._sized(grad_bias_gpu, "grad_bias", (n,), "f32")
        nbytes = lib.tcbnn_linear_grad_workspace_bytes(m, k, n, _lib.DTYPES[self.dtype])
        ws = self._grad_buffer(nbytes)
        self._grad_desc = _lib.LinearGradDesc(
            self.input_gpu.ptr, self.weight_gpu.ptr, _ptr(self.preact_gpu), self.grad_output_gpu.ptr, _ptr(grad_input_gpu),
            _ptr(grad_weight_gpu), _ptr(grad_bias_gpu), m, k, n, _lib.DTYPES[self.dtype], _lib.ACTIVATIONS[self.activation],
            _ld(self.input_gpu), _ld(self.weight_gpu), _ld(self.preact_gpu), _ld(grad_output_gpu), _ld(grad_input_gpu),
            _ld(grad_weight_gpu), _ptr(ws), nbytes)
        self._backward = self._call(lib.tcbnn_linear_backward, self._grad_desc)
        return self

    def get_output_gpu(self):
        return self.output_gpu

    def download_output(self):
        """fp32 [rows][out_features] of a buffer without gaps between rows."""
        return self._download(self.output_gpu, self.rows, self.out_features)


class LayerNormLayerParam(_HeadLayer):
    """output = (input - mean) / sqrt(variance + eps) * gamma + beta over the features of each row."""

    def __init__(self, name, rows, features, dtype="f32", eps=1e-5):
        super().__init__(name, dtype)
        self.rows, self.features, self.eps = rows, features, eps

    def initialize(self, gamma, beta, input_gpu, output_gpu=None, mean_gpu=None, rstd_gpu=None):
        self._forget()
        m, n, dt = self.rows, self.features, self.dtype
        self.input_gpu = self._sized(self._required(input_gpu, "input"), "input", (m, n), dt)
        self.gamma_gpu = self._sized(self._parameter(gamma, "f32", (n,)), "gamma", (n,), "f32")
        self.beta_gpu = self._sized(self._parameter(beta, "f32", (n,)), "beta", (n,), "f32")
        self.output_gpu = self._sized(output_gpu if output_gpu is not None else self._buffer(m * n * ITEMSIZE[dt]), "output", (m, n), dt)
        self.mean_gpu = self._sized(mean_gpu if mean_gpu is not None else self._buffer(4 * m), "mean", (m,), "f32")
        self.rstd_gpu = self._sized(rstd_gpu if rstd_gpu is not None else self._buffer(4 * m), "rstd", (m,), "f32")
        self._desc = _lib.LayerNormDesc(
            self.input_gpu.ptr, _ptr(self.gamma_gpu), _ptr(self.beta_gpu), self.output_gpu.ptr, self.mean_gpu.ptr, self.rstd_gpu.ptr,
            m, n, _lib.DTYPES[self.dtype], self.eps, _ld(self.input_gpu), _ld(self.output_gpu))
        self._forward = self._call(lib.tcbnn_layernorm_forward, self._desc)
        return self

    def initialize_backward(self, grad_output_gpu, grad_input_gpu=None, grad_gamma_gpu=None, grad_beta_gpu=None):
        """After initialize().  Gradients are written where a buffer is given; mean and rstd are those of forward()."""
        m, n, dt = self.rows, self.features, self.dtype
        self.grad_output_gpu = self._sized(self._required(grad_output_gpu, "grad_output"), "grad_output", (m, n), dt)
        self.grad_input_gpu = self._sized(grad_input_gpu, "grad_input", (m, n), dt)
        self.grad_gamma_gpu = self._sized(grad_gamma_gpu, "grad_gamma", (n,), "f32")
        self.grad_beta_gpu = self._sized(grad_beta_gpu, "grad_beta", (n,), "f32")
        nbytes = lib.tcbnn_layernorm_grad_workspace_bytes(m, n)
        ws = self._grad_buffer(nbytes)
        self._grad_desc = _lib.LayerNormGradDesc(
            self.input_gpu.ptr, _ptr(self.gamma_gpu), self.mean_gpu.ptr, self.rstd_gpu.ptr, self.grad_output_gpu.ptr,
            _ptr(grad_input_gpu), _ptr(grad_gamma_gpu), _ptr(grad_beta_gpu), m, n, _lib.DTYPES[self.dtype], _ld(self.input_gpu),
            _ld(grad_output_gpu), _ld(grad_input_gpu), _ptr(ws), nbytes)
        self._backward = self._call(lib.tcbnn_layernorm_backward, self._grad_desc)
        return self

    def get_output_gpu(self):
        return self.output_gpu

    def download_output(self):
        """fp32 [rows][features] of a buffer without gaps between rows."""
        return self._download(self.output_gpu, self.rows, self.features)


class GatedLayerParam(_HeadLayer):
    """output = act(gate) * up with [gate up] = input * weight^T + bias; input [rows][in_features], weight [2 * features]
    [in_features], the gate's rows first, output [rows][features]."""

    def __init__(self, name, rows, in_features, features, dtype="f32", activation="silu"):
        super().__init__(name, dtype)
        if activation not in _lib.ACTIVATIONS:
            raise _lib.TcbnnError("Error: %s: unknown activation %r" % (name, activation))
        self.rows, self.in_features, self.features, self.activation = rows, in_features, features, activation

    def initialize(self, weight, bias, input_gpu, output_gpu=None, preact_gpu=None, save_preact=False):
        """save_preact: keep [gate up], which backward() needs, in a buffer of the layer's own (or give `preact_gpu`,
        [rows][2 * features])."""
        self._forget()
        m, k, n, dt = self.rows, self.in_features, self.features, self.dtype
        self.input_gpu = self._sized(self._required(input_gpu, "input"), "input", (m, k), dt)
        self.weight_gpu = self._sized(self._parameter(self._required(weight, "weight"), dt, (2 * n, k)), "weight", (2 * n, k), dt)
        self.bias_gpu = self._sized(self._parameter(bias, "f32", (2 * n,)), "bias", (2 * n,), "f32")
        self.output_gpu = self._sized(output_gpu if output_gpu is not None else self._buffer(m * n * ITEMSIZE[dt]), "output", (m, n), dt)
        if preact_gpu is None and save_preact:
            preact_gpu = self._buffer(2 * m * n * ITEMSIZE[dt])
        self.preact_gpu = self._sized(preact_gpu, "preact", (m, 2 * n), dt)
        nbytes = lib.tcbnn_gated_workspace_bytes(m, k, n, _lib.DTYPES[dt]) if _anywhere(dt, k, self.input_gpu, self.weight_gpu) else 0
        ws = self._buffer(nbytes) if nbytes else None
        self._desc = _lib.GatedDesc(
            self.input_gpu.ptr, self.weight_gpu.ptr, _ptr(self.bias_gpu), self.output_gpu.ptr, _ptr(self.preact_gpu), m, k, n,
            _lib.DTYPES[dt], _lib.ACTIVATIONS[self.activation], _ld(self.input_gpu), _ld(self.weight_gpu), _ld(self.output_gpu),
            _ld(self.preact_gpu), _ptr(ws), nbytes)
        self._forward = self._call(lib.tcbnn_gated_forward, self._desc)
        return self

    def initialize_backward(self, grad_output_gpu, grad_input_gpu=None, grad_weight_gpu=None, grad_bias_gpu=None):
        """After initialize().  Gradients are written where a buffer is given."""
        m, k, n, dt = self.rows, self.in_features, self.features, self.dtype
        self._required(self.preact_gpu, "preact")
        self.grad_output_gpu = self._sized(self._required(grad_output_gpu, "grad_output"), "grad_output", (m, n), dt)
        self.grad_input_gpu = self._sized(grad_input_gpu, "grad_input", (m, k), dt)
        self.grad_weight_gpu = self._sized(grad_weight_gpu, "grad_weight", (2 * n, k), dt)
        self.grad_bias_gpu = self._sized(grad_bias_gpu, "grad_bias", (2 * n,), "f32")
        nbytes = lib.tcbnn_gated_grad_workspace_bytes(m, k, n, _lib.DTYPES[dt], _anywhere(dt, k, self.input_gpu, self.weight_gpu))
        ws = self._grad_buffer(nbytes)
        self._grad_desc = _lib.GatedGradDesc(
            self.input_gpu.ptr, self.weight_gpu.ptr, self.preact_gpu.ptr, self.grad_output_gpu.ptr, _ptr(grad_input_gpu),
            _ptr(grad_weight_gpu), _ptr(grad_bias_gpu), m, k, n, _lib.DTYPES[dt], _lib.ACTIVATIONS[self.activation],
            _ld(self.input_gpu), _ld(self.weight_gpu), _ld(self.preact_gpu), _ld(grad_output_gpu), _ld(grad_input_gpu),
            _ld(grad_weight_gpu), _ptr(ws), nbytes)
        self._backward = self._call(lib.tcbnn_gated_backward, self._grad_desc)
        return self

    def get_output_gpu(self):
        return self.output_gpu

    def download_output(self):
        """fp32 [rows][features] of a buffer without gaps between rows."""
        return self._download(self.output_gpu, self.rows, self.features)


class BlockNormLayerParam(_HeadLayer):
    """The norms after and before a block, with the residual stream between them:
    new_stream = stream + scale * gate * norm_after(block);  output = norm_before(new_stream).

    `after` and `before` are "rms", "layer" or "none".  Without a block the stream stays as it is (the norm before a first
    block)."""

    def __init__(self, name, rows, features, dtype="f32", after="none", before="rms", scale=1.0, eps=1e-5):
        super().__init__(name, dtype)
        for kind in (after, before):
            if kind not in _lib.NORMS:
                raise _lib.TcbnnError("Error: %s: unknown norm %r" % (name, kind))
        self.rows, self.features, self.after, self.before, self.scale, self.eps = rows, features, after, before, scale, eps

    def initialize(self, stream_gpu, block_gpu=None, gate=None, after_gamma=None, after_beta=None, before_gamma=None,
                   before_beta=None, new_stream_gpu=None, output_gpu=None, after_mean_gpu=None, after_rstd_gpu=None,
                   before_mean_gpu=None, before_rstd_gpu=None):
        """`new_stream_gpu` may be `stream_gpu`.  gate, gammas and betas are fp32 [features]; a beta belongs to a layer norm."""
        self._forget()
        m, n, dt = self.rows, self.features, self.dtype
        self.stream_gpu = self._sized(self._required(stream_gpu, "stream"), "stream", (m, n), dt)
        self.block_gpu = self._sized(block_gpu, "block", (m, n), dt)
        self.gate_gpu, self.after_gamma_gpu, self.after_beta_gpu, self.before_gamma_gpu, self.before_beta_gpu = (
            self._sized(self._parameter(p, "f32", (n,)), what, (n,), "f32")
            for p, what in ((gate, "gate"), (after_gamma, "after_gamma"), (after_beta, "after_beta"),
                            (before_gamma, "before_gamma"), (before_beta, "before_beta")))

        def matrix(buf, what, wanted):
            return self._sized(buf if buf is not None or not wanted else self._buffer(m * n * ITEMSIZE[dt]), what, (m, n), dt)

        def statistic(buf, what, wanted):
            return self._sized(buf if buf is not None or not wanted else self._buffer(4 * m), what, (m,), "f32")

        written = matrix(new_stream_gpu, "new_stream", block_gpu is not None)
        self.new_stream_gpu = self.stream_gpu if written is None else written
        self.output_gpu = matrix(output_gpu, "output", self.before != "none")
        self.after_mean_gpu = statistic(after_mean_gpu, "after_mean", self.after == "layer")
        self.after_rstd_gpu = statistic(after_rstd_gpu, "after_rstd", self.after != "none")
        self.before_mean_gpu = statistic(before_mean_gpu, "before_mean", self.before == "layer")
        self.before_rstd_gpu = statistic(before_rstd_gpu, "before_rstd", self.before != "none")
        self._desc = _lib.BlockNormDesc(
            self.stream_gpu.ptr, _ptr(self.block_gpu), _ptr(self.gate_gpu), _ptr(self.after_gamma_gpu), _ptr(self.after_beta_gpu),
            _ptr(self.before_gamma_gpu), _ptr(self.before_beta_gpu), _ptr(written), _ptr(self.output_gpu), _ptr(self.after_mean_gpu),
            _ptr(self.after_rstd_gpu), _ptr(self.before_mean_gpu), _ptr(self.before_rstd_gpu), m, n, _lib.DTYPES[dt],
            _lib.NORMS[self.after], _lib.NORMS[self.before], self.scale, self.eps, _ld(self.stream_gpu), _ld(self.block_gpu),
            _ld(written), _ld(self.output_gpu))
        self._forward = self._call(lib.tcbnn_blocknorm_forward, self._desc)
        return self

    def initialize_backward(self, grad_output_gpu=None, grad_new_stream_gpu=None, grad_stream_gpu=None, grad_block_gpu=None,
                            grad_gate_gpu=None, grad_after_gamma_gpu=None, grad_after_beta_gpu=None, grad_before_gamma_gpu=None,
                            grad_before_beta_gpu=None):
        """After initialize().  Of the first two, None counts as 0; the other gradients are written where a buffer is given.
        The new stream and the statistics are those of forward()."""
        m, n, dt = self.rows, self.features, self.dtype
        self.grad_output_gpu, self.grad_new_stream_gpu, self.grad_stream_gpu, self.grad_block_gpu = (
            self._sized(buf, what, (m, n), dt)
            for buf, what in ((grad_output_gpu, "grad_output"), (grad_new_stream_gpu, "grad_new_stream"),
                              (grad_stream_gpu, "grad_stream"), (grad_block_gpu, "grad_block")))
        self.grad_gate_gpu, self.grad_after_gamma_gpu, self.grad_after_beta_gpu, self.grad_before_gamma_gpu, self.grad_before_beta_gpu = (
            self._sized(buf, what, (n,), "f32")
            for buf, what in ((grad_gate_gpu, "grad_gate"), (grad_after_gamma_gpu, "grad_after_gamma"),
                              (grad_after_beta_gpu, "grad_after_beta"), (grad_before_gamma_gpu, "grad_before_gamma"),
                              (grad_before_beta_gpu, "grad_before_beta")))
        nbytes = lib.tcbnn_blocknorm_grad_workspace_bytes(m, n, _lib.DTYPES[dt])
        ws = self._grad_buffer(nbytes)
        self._grad_desc = _lib.BlockNormGradDesc(
            self.new_stream_gpu.ptr, _ptr(self.block_gpu), _ptr(self.gate_gpu), _ptr(self.after_gamma_gpu), _ptr(self.after_beta_gpu),
            _ptr(self.before_gamma_gpu), _ptr(self.after_mean_gpu), _ptr(self.after_rstd_gpu), _ptr(self.before_mean_gpu),
            _ptr(self.before_rstd_gpu), _ptr(grad_output_gpu), _ptr(grad_new_stream_gpu), _ptr(grad_stream_gpu), _ptr(grad_block_gpu),
            _ptr(grad_gate_gpu), _ptr(grad_after_gamma_gpu), _ptr(grad_after_beta_gpu), _ptr(grad_before_gamma_gpu),
            _ptr(grad_before_beta_gpu), m, n, _lib.DTYPES[dt], _lib.NORMS[self.after], _lib.NORMS[self.before], self.scale,
            _ld(self.new_stream_gpu), _ld(self.block_gpu), _ld(grad_output_gpu), _ld(grad_new_stream_gpu), _ld(grad_stream_gpu),
            _ld(grad_block_gpu), _ptr(ws), nbytes)
        self._backward = self._call(lib.tcbnn_blocknorm_backward, self._grad_desc)
        return self

    def get_output_gpu(self):
        return self.output_gpu

    def download_output(self):
        """fp32 [rows][features] of a buffer without gaps between rows."""
        return self._download(self._required(self.output_gpu, "output"), self.rows, self.features)


class LogProbsLayerParam(_HeadLayer):
    """Of every row of logits: log probability and rank of a given class, entropy, the `top` best classes."""

    def __init__(self, name, rows, classes, top=0, dtype="f32"):
        super().__init__(name, dtype)
        self.rows, self.classes, self.top = rows, classes, top

    def initialize(self, logits_gpu, targets_gpu=None, logprob_gpu=None, entropy_gpu=None, logsumexp_gpu=None, rank_gpu=None,
                   top_index_gpu=None, top_logprob_gpu=None):
        """Without `targets_gpu` (int32, -1: none) no log probabilities and ranks of given classes are computed."""
        self._forget()
        m, n, k = self.rows, self.classes, self.top
        self.logits_gpu = self._sized(self._required(logits_gpu, "logits"), "logits", (m, n), self.dtype)
        self.targets_gpu = self._sized(targets_gpu, "targets", (m,), "i32")

        def out(buf, what, shape, wanted=True, dtype="f32"):
            return self._sized(buf if buf is not None or not wanted else self._buffer(4 * int(np.prod(shape))), what, shape, dtype, gaps=False)

        given = targets_gpu is not None
        self.logprob_gpu = out(logprob_gpu, "logprob", (m,), given)
        self.entropy_gpu = out(entropy_gpu, "entropy", (m,))
        self.logsumexp_gpu = out(logsumexp_gpu, "logsumexp", (m,))
        self.rank_gpu = out(rank_gpu, "rank", (m,), given, "i32")
        self.top_index_gpu = out(top_index_gpu, "top_index", (m, k), k > 0, "i32")
        self.top_logprob_gpu = out(top_logprob_gpu, "top_logprob", (m, k), k > 0)
        nbytes = lib.tcbnn_logprobs_workspace_bytes(m, n, k, _lib.DTYPES[self.dtype])
        ws = self._buffer(nbytes) if nbytes else None
        self._desc = _lib.LogProbsDesc(
            self.logits_gpu.ptr, _ptr(targets_gpu), _ptr(self.logprob_gpu), _ptr(self.entropy_gpu), _ptr(self.logsumexp_gpu),
            _ptr(self.rank_gpu), _ptr(self.top_index_gpu), _ptr(self.top_logprob_gpu), m, n, k, _lib.DTYPES[self.dtype],
            _ld(self.logits_gpu), _ptr(ws), nbytes)
        self._forward = self._call(lib.tcbnn_logprobs_forward, self._desc)
        return self

    def initialize_backward(self, grad_logprob_gpu, grad_entropy_gpu, grad_logits_gpu):
        """After initialize(); either of the first two may be None.  logsumexp and entropy are those of forward()."""
        m, n = self.rows, self.classes
        if grad_logprob_gpu is not None:
            self._required(self.targets_gpu, "targets")
        self.grad_logprob_gpu = self._sized(grad_logprob_gpu, "grad_logprob", (m,), "f32")
        self.grad_entropy_gpu = self._sized(grad_entropy_gpu, "grad_entropy", (m,), "f32")
        self.grad_logits_gpu = self._sized(self._required(grad_logits_gpu, "grad_logits"), "grad_logits", (m, n), self.dtype)
        self._grad_desc = _lib.LogProbsGradDesc(
            self.logits_gpu.ptr, _ptr(self.targets_gpu), self.logsumexp_gpu.ptr, self.entropy_gpu.ptr, _ptr(grad_logprob_gpu),
            _ptr(grad_entropy_gpu), grad_logits_gpu.ptr, m, n, _lib.DTYPES[self.dtype], _ld(self.logits_gpu), _ld(grad_logits_gpu))
        self._backward = self._call(lib.tcbnn_logprobs_backward, self._grad_desc)
        return self

    def download_output(self):
        """dict of the host arrays of what forward() wrote."""
        m, k = self.rows, self.top
        out = {"entropy": self.entropy_gpu.to_numpy(np.float32, (m,)), "logsumexp": self.logsumexp_gpu.to_numpy(np.float32, (m,))}
        if self.targets_gpu is not None:
            out["logprob"] = self.logprob_gpu.to_numpy(np.float32, (m,))
            out["rank"] = self.rank_gpu.to_numpy(np.int32, (m,))
        if k:
            out["top_index"] = self.top_index_gpu.to_numpy(np.int32, (m, k))
            out["top_logprob"] = self.top_logprob_gpu.to_numpy(np.float32, (m, k))
        return out


class LinearLossLayerParam(_HeadLayer):
    """loss = logsumexp(z) - z[target] of every row of z = input * weight^T + bias: the softmax cross entropy of a linear
    classifier that keeps no logits; input [rows][in_features], weight [classes][in_features]."""

    def __init__(self, name, rows, in_features, classes, dtype="f32"):
        super().__init__(name, dtype)
        self.rows, self.in_features, self.classes = rows, in_features, classes

    def initialize(self, weight, bias, input_gpu, targets_gpu, loss_gpu=None, logsumexp_gpu=None, logsumexp_rest_gpu=None):
        """targets: int32 [rows], -1 for rows without a class (loss 0, no gradient).  logsumexp_rest: what rounding left of
        logsumexp, for backward()."""
        self._forget()
        m, k, n, dt = self.rows, self.in_features, self.classes, self.dtype
        self.input_gpu = self._sized(self._required(input_gpu, "input"), "input", (m, k), dt)
        self.weight_gpu = self._sized(self._parameter(self._required(weight, "weight"), dt, (n, k)), "weight", (n, k), dt)
        self.bias_gpu = self._sized(self._parameter(bias, "f32", (n,)), "bias", (n,), "f32")
        self.targets_gpu = self._sized(self._required(targets_gpu, "targets"), "targets", (m,), "i32")
        self.loss_gpu, self.logsumexp_gpu, self.logsumexp_rest_gpu = (
            self._sized(buf if buf is not None else self._buffer(4 * m), what, (m,), "f32")
            for buf, what in ((loss_gpu, "loss"), (logsumexp_gpu, "logsumexp"), (logsumexp_rest_gpu, "logsumexp_rest")))
        nbytes = lib.tcbnn_linear_loss_workspace_bytes(m, k, n, _lib.DTYPES[dt], _anywhere(dt, k, self.input_gpu, self.weight_gpu))
        ws = self._buffer(nbytes) if nbytes else None
        self._desc = _lib.LinearLossDesc(
            self.input_gpu.ptr, self.weight_gpu.ptr, _ptr(self.bias_gpu), self.targets_gpu.ptr, self.loss_gpu.ptr,
            self.logsumexp_gpu.ptr, m, k, n, _lib.DTYPES[dt], _ld(self.input_gpu), _ld(self.weight_gpu), _ptr(ws), nbytes,
            self.logsumexp_rest_gpu.ptr)
        self._forward = self._call(lib.tcbnn_linear_loss_forward, self._desc)
        return self

    def initialize_backward(self, grad_loss_gpu, grad_input_gpu=None, grad_weight_gpu=None, grad_bias_gpu=None):
        """After initialize().  grad_loss: fp32 [rows] (1 / n for the mean of n rows).  Gradients are written where a buffer is
        given; loss, logsumexp and its rest are those of forward()."""
        m, k, n, dt = self.rows, self.in_features, self.classes, self.dtype
        self.grad_loss_gpu = self._sized(self._required(grad_loss_gpu, "grad_loss"), "grad_loss", (m,), "f32")
        self.grad_input_gpu = self._sized(grad_input_gpu, "grad_input", (m, k), dt)
        self.grad_weight_gpu = self._sized(grad_weight_gpu, "grad_weight", (n, k), dt)
        self.grad_bias_gpu = self._sized(grad_bias_gpu, "grad_bias", (n,), "f32")
        nbytes = lib.tcbnn_linear_loss_grad_workspace_bytes(m, k, n, _lib.DTYPES[dt], _anywhere(dt, k, self.input_gpu, self.weight_gpu))
        ws = self._grad_buffer(nbytes)
        self._grad_desc = _lib.LinearLossGradDesc(
            self.input_gpu.ptr, self.weight_gpu.ptr, _ptr(self.bias_gpu), self.targets_gpu.ptr, self.logsumexp_gpu.ptr,
            self.loss_gpu.ptr, self.grad_loss_gpu.ptr, _ptr(grad_input_gpu), _ptr(grad_weight_gpu), _ptr(grad_bias_gpu), m, k, n, _lib.DTYPES[dt],
            _ld(self.input_gpu), _ld(self.weight_gpu), _ld(grad_input_gpu), _ld(grad_weight_gpu), _ptr(ws), nbytes,
            self.logsumexp_rest_gpu.ptr)
        self._backward = self._call(lib.tcbnn_linear_loss_backward, self._grad_desc)
        return self

    def download_output(self):
        """dict of the host arrays of what forward() wrote."""
        return {"loss": self.loss_gpu.to_numpy(np.float32, (self.rows,)), "logsumexp": self.logsumexp_gpu.to_numpy(np.float32, (self.rows,))}


class _Head:
    """What heads share: `params` (fp32 host arrays by name, those of weights beginning with w), `_devices` and `_grads` (their buffers and
    their gradients' by the same names), `layers` in the order that forward() takes them."""

    def forward(self, stream=None):
        for layer in self.layers:
            layer.forward(stream)

    def backward(self, stream=None):
        """The gradients of all parameters, of the mean cross entropy of the last forward()."""
        for layer in reversed(self.layers):
            layer.backward(stream)

    def gradients(self):
        """fp32 host arrays of the last backward()'s gradients, by parameter."""
        _lib.device_synchronize()
        out = {}
        for name, a in self.params.items():
            dt = self.dtype if name[0] == "w" else "f32"
            out[name] = decode(self._grads[name].to_numpy(storage(dt), a.shape), dt)
        return out

    def step(self, rate):
        for name, g in self.gradients().items():
            self.params[name] -= np.float32(rate) * g
            self._devices[name].upload(encode(self.params[name], self.dtype if name[0] == "w" else "f32"))


class FloatHead(_Head):
    """A float head on `features` values a row, as on the last binary layer of a network:
    norm -> linear (GELU), + the features where there are as many hidden values -> norm -> linear -> log probabilities of
    `classes`.  The features are given (the network below them is frozen): they get no gradient.

    forward() scores the rows' targets and ranks the best classes; backward() leaves the gradient of the mean cross
    entropy in the layers' gradient buffers; step() takes a step of gradient descent on the parameters, which are kept
    in fp32 on the host."""

    def __init__(self, rows, features, hidden, classes, dtype="f32", top=5):
        self.rows, self.features, self.hidden, self.classes, self.dtype = rows, features, hidden, classes, dtype
        self.norm1 = LayerNormLayerParam("Norm1", rows, features, dtype)
        self.linear1 = LinearLayerParam("Linear1", rows, features, hidden, dtype, "gelu")
        self.norm2 = LayerNormLayerParam("Norm2", rows, hidden, dtype)
        self.linear2 = LinearLayerParam("Linear2", rows, hidden, classes, dtype)
        self.logprobs = LogProbsLayerParam("LogProbs", rows, classes, min(top, classes), dtype)
        self.layers = [self.norm1, self.linear1, self.norm2, self.linear2, self.logprobs]

    def initialize(self, features_gpu, targets, seed=0):
        """features_gpu: [rows][features] in the head's dtype; targets: int32 [rows], -1 for rows without a class."""
        if np.size(targets) != self.rows:
            raise _lib.TcbnnError("Error: %d targets for %d rows" % (np.size(targets), self.rows))
        rng = np.random.default_rng(seed)
        k, h, c, m = self.features, self.hidden, self.classes, self.rows
        self.params = {"gamma1": np.ones(k, np.float32), "beta1": np.zeros(k, np.float32),
                       "w1": rng.normal(0, k ** -0.5, (h, k)).astype(np.float32), "b1": np.zeros(h, np.float32),
                       "gamma2": np.ones(h, np.float32), "beta2": np.zeros(h, np.float32),
                       "w2": rng.normal(0, h ** -0.5, (c, h)).astype(np.float32), "b2": np.zeros(c, np.float32)}
        p, size = self.params, 4 if self.dtype == "f32" else 2
        targets = np.ascontiguousarray(targets, np.int32)
        n1, l1, n2, l2, lp = self.layers
        n1.initialize(p["gamma1"], p["beta1"], features_gpu)
        l1.initialize(p["w1"], p["b1"], n1.output_gpu, residual_gpu=features_gpu if h == k else None, save_preact=True)
        n2.initialize(p["gamma2"], p["beta2"], l1.output_gpu)
        l2.initialize(p["w2"], p["b2"], n2.output_gpu)
        self._targets = DeviceBuffer.from_numpy(targets)
        lp.initialize(l2.output_gpu, self._targets)
        self._grads = {name: DeviceBuffer(a.size * (size if name[0] == "w" else 4)) for name, a in p.items()}
        self._flows = [DeviceBuffer(m * n * size) for n in (c, h, h, k)]
        g = self._grads
        given = max(1, int((targets >= 0).sum()))
        self._loss = DeviceBuffer.from_numpy(np.where(targets >= 0, np.float32(-1.0 / given), np.float32(0)))
        self._given = given
        lp.initialize_backward(self._loss, None, self._flows[0])
        l2.initialize_backward(self._flows[0], self._flows[1], g["w2"], g["b2"])
        n2.initialize_backward(self._flows[1], self._flows[2], g["gamma2"], g["beta2"])
        l1.initialize_backward(self._flows[2], self._flows[3], g["w1"], g["b1"])
        n1.initialize_backward(self._flows[3], None, g["gamma1"], g["beta1"])
        self._devices = {"gamma1": n1.gamma_gpu, "beta1": n1.beta_gpu, "w1": l1.weight_gpu, "b1": l1.bias_gpu,
                         "gamma2": n2.gamma_gpu, "beta2": n2.beta_gpu, "w2": l2.weight_gpu, "b2": l2.bias_gpu}
        return self

    def loss(self):
        """The mean cross entropy of the last forward()."""
        _lib.device_synchronize()
        return -float(self.logprobs.logprob_gpu.to_numpy(np.float32, (self.rows,)).astype(np.float64).sum()) / self._given

    def release(self):
        for layer in self.layers:
            layer.release()
        for buf in [self._targets, self._loss] + self._flows + list(self._grads.values()):
            buf.free()


class GatedHead(_Head):
    """A float head of gated residual blocks on `features` values a row:
    norm -> [gated product (SiLU) -> linear, normed, gated and added to the stream, norm] x blocks -> linear loss over `classes`,
    with RMS norms.  The features are given (the network below them is frozen): they get no gradient.

    forward() computes the rows' losses, without logits; backward() leaves the gradient of the mean cross entropy in the layers' gradient
    buffers; step() takes a step of gradient descent; score() ranks the best classes of the last forward()."""

    def __init__(self, rows, features, hidden, classes, dtype="f32", blocks=1, scale=0.5, top=5):
        if blocks < 1:
            raise _lib.TcbnnError("Error: a gated head of %d blocks" % blocks)
        self.rows, self.features, self.hidden, self.classes, self.dtype, self.blocks = rows, features, hidden, classes, dtype, blocks
        self.norm = BlockNormLayerParam("Norm", rows, features, dtype)
        self.gated = [GatedLayerParam("Gated%d" % i, rows, features, hidden, dtype) for i in range(blocks)]
        self.down = [LinearLayerParam("Down%d" % i, rows, hidden, features, dtype) for i in range(blocks)]
        self.norms = [BlockNormLayerParam("Norms%d" % i, rows, features, dtype, after="rms", scale=scale) for i in range(blocks)]
        self.linear_loss = LinearLossLayerParam("Loss", rows, features, classes, dtype)
        self.classifier = LinearLayerParam("Classifier", rows, features, classes, dtype)
        self.logprobs = LogProbsLayerParam("LogProbs", rows, classes, min(top, classes), dtype)
        self.layers = [self.norm]
        for block in zip(self.gated, self.down, self.norms):
            self.layers += block
        self.layers.append(self.linear_loss)
        self._score = None

    def initialize(self, features_gpu, targets, seed=0):
        """features_gpu: [rows][features] in the head's dtype; targets: int32 [rows], -1 for rows without a class."""
        if np.size(targets) != self.rows:
            raise _lib.TcbnnError("Error: %d targets for %d rows" % (np.size(targets), self.rows))
        rng = np.random.default_rng(seed)
        k, h, c, m, size = self.features, self.hidden, self.classes, self.rows, 4 if self.dtype == "f32" else 2

        def weight(out, inp):
            return rng.normal(0, inp ** -0.5, (out, inp)).astype(np.float32)

        p = self.params = {"gamma": np.ones(k, np.float32)}
        for i in range(self.blocks):
            p.update({"w_gated%d" % i: weight(2 * h, k), "b_gated%d" % i: np.zeros(2 * h, np.float32), "w_down%d" % i: weight(k, h),
                      "gate%d" % i: np.ones(k, np.float32), "gamma_after%d" % i: np.ones(k, np.float32),
                      "gamma_before%d" % i: np.ones(k, np.float32)})
        p.update({"w_class": weight(c, k), "b_class": np.zeros(c, np.float32)})
        targets = np.ascontiguousarray(targets, np.int32)
        self._given = max(1, int((targets >= 0).sum()))
        self._targets = DeviceBuffer.from_numpy(targets)
        self._loss = DeviceBuffer.from_numpy(np.where(targets >= 0, np.float32(1.0 / self._given), np.float32(0)))
        g = self._grads = {name: DeviceBuffer(a.size * (size if name[0] == "w" else 4)) for name, a in p.items()}
        self._flows = []

        def flow(cols):
            self._flows.append(DeviceBuffer(m * cols * size))
            return self._flows[-1]

        self.norm.initialize(features_gpu, before_gamma=p["gamma"])
        stream, y = features_gpu, self.norm.output_gpu
        for i, (gated, down, norms) in enumerate(zip(self.gated, self.down, self.norms)):
            gated.initialize(p["w_gated%d" % i], p["b_gated%d" % i], y, save_preact=True)
            down.initialize(p["w_down%d" % i], None, gated.output_gpu)
            norms.initialize(stream, down.output_gpu, gate=p["gate%d" % i], after_gamma=p["gamma_after%d" % i], before_gamma=p["gamma_before%d" % i])
            stream, y = norms.new_stream_gpu, norms.output_gpu
        self.linear_loss.initialize(p["w_class"], p["b_class"], y, self._targets)
        d_y, d_stream = flow(k), None
        self.linear_loss.initialize_backward(self._loss, d_y, g["w_class"], g["b_class"])
        for i in reversed(range(self.blocks)):
            d_block, d_hidden, before = flow(k), flow(h), flow(k) if i else None  # (the features get no gradient)
            self.norms[i].initialize_backward(d_y, d_stream, before, d_block, g["gate%d" % i], g["gamma_after%d" % i],
                                              grad_before_gamma_gpu=g["gamma_before%d" % i])
            self.down[i].initialize_backward(d_block, d_hidden, g["w_down%d" % i])
            d_y = flow(k)
            self.gated[i].initialize_backward(d_hidden, d_y, g["w_gated%d" % i], g["b_gated%d" % i])
            d_stream = before
        self.norm.initialize_backward(d_y, grad_before_gamma_gpu=g["gamma"])
        self._devices = {"gamma": self.norm.before_gamma_gpu, "w_class": self.linear_loss.weight_gpu, "b_class": self.linear_loss.bias_gpu}
        for i in range(self.blocks):
            self._devices.update({"w_gated%d" % i: self.gated[i].weight_gpu, "b_gated%d" % i: self.gated[i].bias_gpu,
                                  "w_down%d" % i: self.down[i].weight_gpu, "gate%d" % i: self.norms[i].gate_gpu,
                                  "gamma_after%d" % i: self.norms[i].after_gamma_gpu, "gamma_before%d" % i: self.norms[i].before_gamma_gpu})
        self._score = None
        return self

    def loss(self):
        """The mean cross entropy of the last forward()."""
        _lib.device_synchronize()
        return float(self.linear_loss.loss_gpu.to_numpy(np.float32, (self.rows,)).astype(np.float64).sum()) / self._given

    def score(self, stream=None):
        """Log probabilities, ranks and best classes of the last forward()'s rows (LogProbsLayerParam's outputs): with logits, which the
        first call makes room for."""
        if self._score is None:
            last = self.linear_loss
            self.classifier.initialize(last.weight_gpu, last.bias_gpu, last.input_gpu)
            self.logprobs.initialize(self.classifier.output_gpu, self._targets)
            self._score = [self.classifier, self.logprobs]
        for layer in self._score:
            layer.forward(stream)
        _lib.device_synchronize()
        return self.logprobs.download_output()

    def release(self):
        for layer in self.layers + [self.classifier, self.logprobs]:
            layer.release()
        for buf in [self._targets, self._loss] + self._flows + list(self._grads.values()):
            buf.free()
