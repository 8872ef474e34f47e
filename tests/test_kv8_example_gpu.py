"""examples/kv8_decode.py: the operators of the 8-bit cache together with the projections, against the same layer in 64 bits.

The reference keeps k and v as they are, so the difference is the cache's: an element is off by at most half a step of its page
(the largest magnitude of 16 tokens of a head / 127) for its store and as much for each growth of the scale that follows. With
at most 16 stores to a page and magnitudes of one size, a few half steps of about 3.5 / 127 sigma are about 2 % of
sigma an element, independent from element to element; scores and outputs average them. The bound is 5 % of the
reference's norm; without the rotation, the norms or the mask the difference is of the order of the norm itself.
"""
import os
import sys

import numpy as np
import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


def reference(layer, xs):
    """Outputs of one sequence in 64 bits: xs [tokens][hidden]."""
    w = {n: torch.from_numpy(t.dequant_host().reshape(t.rows, t.cols)).double().cuda() for n, t in layer.w.items()}
    h, kvh, hd = layer.heads, layer.kvh, layer.hd
    qkv = (xs.double() @ w["qkv"].T).view(-1, h + 2 * kvh, hd)
    c, s = layer.table.double()[: len(xs)][:, None].unbind(-1)

    def turn(x, norm):
        x = x / (x.pow(2).mean(-1, keepdim=True) + 1e-5).sqrt() * norm.double()
        a, b = x[..., 0::2], x[..., 1::2]
        return torch.stack([a * c - b * s, a * s + b * c], -1).flatten(-2)

    q, k, v = turn(qkv[:, :h], layer.q_norm), turn(qkv[:, h:h + kvh], layer.k_norm), qkv[:, h + kvh:]
    k, v = (t.repeat_interleave(h // kvh, 1) for t in (k, v))
    z = torch.einsum("thd,shd->hts", q, k) / hd ** 0.5
    z = z.masked_fill(torch.ones(len(xs), len(xs), device="cuda").triu(1).bool(), float("-inf"))
    return torch.einsum("hts,shd->thd", z.softmax(-1), v).flatten(1) @ w["o"].T


def test_the_example_layer_follows_the_formula():
    sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples"))
    import kv8_decode

    prompts, steps = (100, 7, 33), 24
    out, outs, us, layer = kv8_decode.run(prompts, steps)
    torch.cuda.synchronize()
    g = torch.Generator(device="cuda").manual_seed(0)
    x = torch.empty(sum(prompts), layer.hidden, device="cuda").normal_(generator=g)
    starts = np.concatenate([[0], np.cumsum(prompts)])
    for s, n in enumerate(prompts):
        a, b = starts[s], starts[s + 1]
        norm = lambda t: torch.nn.functional.normalize(t) * layer.hidden ** 0.5  # noqa: E731
        xs = torch.cat([x[a:b], out[b - 1:b], norm(outs[:-1, s])])  # what the layer was fed
        ref = reference(layer, xs)
        for got, want in ((out[a:b].double(), ref[:n]), (outs[:, s].double(), ref[n:])):
            assert float((got - want).norm() / want.norm()) < 0.05
    assert us > 0
