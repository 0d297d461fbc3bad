"""A float head on the frozen binary layers of the MLP (In -> Fc x 3 of mnist_mlp_spec): trained for a few steps on synthetic
labels, then used to score a batch.

    python -m tcbnn_amd.head_example [--batch 1024] [--hidden 1024] [--classes 10] [--steps 40] [--rate 0.02] [--dtype f32]
                                      [--head float|gated] [--blocks 1]

--head gated takes gated residual blocks and a loss that keeps no logits in place of the two linear layers.

The labels are those of a random linear rule on the images, so the loss falls from log(classes)."""
import argparse

import numpy as np

from . import _lib, nets
from ._lib import check, lib
from .device import DeviceBuffer
from .head import FloatHead, GatedHead, encode


def binary_features(batch, width=1024, seed=0):
    """The +-1 outputs of the MLP's last hidden layer for a synthetic batch, fp32 [batch][width] on the device, the images, and
    the layers that made them."""
    spec = nets.mnist_mlp_spec(batch=batch, n_hidden=width)[:-1]
    images = nets.synthetic_input(spec, seed)
    trunk = nets.Network(spec, nets.synthetic_weights(spec, seed), images)
    trunk.forward()
    features = DeviceBuffer(4 * batch * width)
    check(lib.tcbnn_unpack_fc_output(trunk.order[-1].get_output_gpu().ptr, features.ptr, batch, width, None))
    return features, images, trunk


def main(argv=None):
    ap = argparse.ArgumentParser(description=__doc__.split("\n\n")[0])
    ap.add_argument("--batch", type=int, default=1024)
    ap.add_argument("--hidden", type=int, default=1024)
    ap.add_argument("--classes", type=int, default=10)
    ap.add_argument("--steps", type=int, default=40)
    ap.add_argument("--rate", type=float, default=0.02)
    ap.add_argument("--dtype", choices=sorted(_lib.DTYPES), default="f32")
    ap.add_argument("--head", choices=["float", "gated"], default="float")
    ap.add_argument("--blocks", type=int, default=1)
    a = ap.parse_args(argv)
    features, images, trunk = binary_features(a.batch, a.hidden)
    rule = np.random.default_rng(1).standard_normal((images.shape[1], a.classes)).astype(np.float32)
    targets = (images @ rule).argmax(1).astype(np.int32)
    if a.dtype != "f32":  # +-1 is exact in every type
        bits = encode(features.to_numpy(np.float32, (a.batch, a.hidden)), a.dtype)
        features = DeviceBuffer.from_numpy(bits)
    if a.head == "gated":
        head = GatedHead(a.batch, a.hidden, a.hidden, a.classes, a.dtype, a.blocks).initialize(features, targets)
    else:
        head = FloatHead(a.batch, a.hidden, a.hidden, a.classes, a.dtype).initialize(features, targets)
    losses = []
    for step in range(a.steps + 1):
        head.forward()
        losses.append(head.loss())
        if step < a.steps:
            head.backward()
            head.step(a.rate)
    scores = head.score() if a.head == "gated" else head.logprobs.download_output()
    k = head.logprobs.top
    print("loss %.4f -> %.4f in %d steps; top-1 %.1f %%, top-%d %.1f %%, mean entropy %.3f nats" % (
        losses[0], losses[-1], a.steps, 100 * (scores["rank"] == 0).mean(), k, 100 * (scores["rank"] < k).mean(),
        scores["entropy"].mean()))
    print("image 0: label %d; best classes %s, log probabilities %s" % (
        targets[0], scores["top_index"][0].tolist(), np.round(scores["top_logprob"][0], 3).tolist()))
    head.release()
    trunk.release()
    return losses


if __name__ == "__main__":
    main()
