"""The floating point end of a network: linear layers, layer norms and log probabilities, forward and backward.

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


class FloatHead:
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

    def forward(self, stream=None):
        for layer in self.layers:
            layer.forward(stream)

    def backward(self, stream=None):
        """The gradients of all parameters, of the mean cross entropy of the last forward()."""
        for layer in reversed(self.layers):
            layer.backward(stream)

    def loss(self):
        """The mean cross entropy of the last forward()."""
        _lib.device_synchronize()
        return -float(self.logprobs.logprob_gpu.to_numpy(np.float32, (self.rows,)).astype(np.float64).sum()) / self._given

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

    def release(self):
        for layer in self.layers:
            layer.release()
        for buf in [self._targets, self._loss] + self._flows + list(self._grads.values()):
            buf.free()
