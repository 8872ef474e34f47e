"""How far attention over the 8-bit cache may be off in norm, against the outputs' own size.

Queries and values are independent normal values, so an output is a random walk over its context: sum p_t v_t of n
tokens is sqrt(n) smaller than the sum of magnitudes, and an error of a token's own size does not hide in it.
Bounds are of the norm over all outputs, relative to the norm of the outputs:
  * rounding to the rows' type: measured on the 64-bit result itself;
  * p rounded to 11 bits (16-bit rows other than f16 with at most 8 rows of a kv head): each p is off by at most 2^-11
    of itself, 2^-11 / sqrt(3) in the root mean square at most, independently of v, so that the walk is off by as much;
  * f32 arithmetic: a score u = s + log2 b of 8 to 16 is rounded to 2^-20 / sqrt(12) = 2.8e-7 (root mean square, times
    ln 2), its products carry about 2e-7, the exponential 2^-22.5, sums of the pages' products at most 1024 roundings
    to nearest of 2^-24 / sqrt(3) each (1.1e-6 at 131072 tokens of one warp set). Together below 1.3e-6; the bound is
    2^-18.
  * f32 rows over ordinary contexts (unit normal queries, scores of about 1): the rounding of u, then of 4 to 8, is
    1e-7, the second terms of q leave 2^-23 / sqrt(3) of a score, the tensor core cuts off 2^-24 of it on average in
    each of at most 8 steps (3e-7 if all of them point the same way), the exponential 2^-22.5 / sqrt(3). Together
    0.4e-6; the bound is 1.2e-6. Products without the second terms are off by 2^-12: the last test makes sure of it.
These add up as squares (they are independent); 1 % is left for their random correlation.
"""
import math

import pytest

from paraoxidizer_b200 import _lib as L
from paraoxidizer_b200.backend import CudaBackend

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

PAGE = 16
STREAM = 1
TYPES = {"f32": (torch.float32, L.POX_F32), "f16": (torch.float16, L.POX_F16), "bf16": (torch.bfloat16, L.POX_BF16)}


@pytest.fixture(scope="module")
def be():
    b = CudaBackend.create(0)
    yield b
    b.synchronize()
    b.close()


class Shared:
    """`seqs` sequences of one context whose block tables name the same pages (a shared prefix: reading it is all that
    attention does), so that long contexts of many sequences need little memory."""

    def __init__(self, seqs, rows, ctx, heads, kvh, hd, dtype, seed=1):
        dt, code = TYPES[dtype]
        g = torch.Generator(device="cuda").manual_seed(seed)
        nb = (ctx + PAGE - 1) // PAGE
        self.hd, self.ctx, self.group, self.rows = hd, ctx, heads // kvh, rows
        x = torch.randn(nb, kvh, 32 * hd, generator=g, device="cuda") * 36
        self.pages = x.round().clamp(-127, 127).to(torch.int8)
        self.scales = (torch.rand(nb, kvh, 2, generator=g, device="cuda") * 0.6).exp() * 0.02
        self.tab = torch.randperm(nb, generator=g, device="cuda").int()[None].repeat(seqs, 1).contiguous()
        self.starts = torch.arange(seqs + 1, device="cuda", dtype=torch.int32) * rows
        self.lens = torch.full((seqs,), ctx, device="cuda", dtype=torch.int32)
        self.q = torch.randn(seqs * rows, heads, hd, generator=g, device="cuda").to(dt)
        self.out = torch.empty_like(self.q)
        self.cache = L.Kv8Cache(self.pages.data_ptr(), self.scales.data_ptr(), nb, kvh, hd)
        self.batch = L.Kv8Batch(self.starts.data_ptr(), self.lens.data_ptr(), self.tab.data_ptr(), seqs, seqs * rows,
                                rows, ctx, nb)
        self.view = lambda t: L.Rows(t.data_ptr(), code, t.stride(0), t.stride(1))

    def attend(self, be):
        be.kv8_attention(self.cache, self.batch, self.view(self.q), self.view(self.out), self.q.shape[1], 0.0, STREAM)
        be.synchronize()
        return self.out.double()

    def values(self, side, h):
        t, d = torch.meshgrid(torch.arange(PAGE, device="cuda"), torch.arange(self.hd, device="cuda"), indexing="ij")
        hd = self.hd
        at = 16 * hd + 16 * d + t if side else t * hd + (d ^ (64 * (t % 2)) if hd == 128 else d)
        ids = self.tab[0].long()
        x = self.pages[ids][:, h][:, at].double() * self.scales[ids][:, h, side, None, None].double()
        return x.reshape(-1, hd)[: self.ctx]

    def formula(self, q_term=lambda x: x, p_term=lambda x: x):
        """The definition in 64 bits; q_term and p_term stand for roundings of q and of p before their products."""
        q = q_term(self.q).double()
        ref = torch.empty_like(q)
        last = torch.arange(q.shape[0], device="cuda") % self.rows + self.ctx - self.rows
        for h in range(q.shape[1]):
            k, v = self.values(0, h // self.group), self.values(1, h // self.group)
            for r in range(0, q.shape[0], 256):
                z = q[r:r + 256, h] @ k.T / self.hd ** 0.5
                z.masked_fill_(torch.arange(self.ctx, device="cuda") > last[r:r + 256, None], -math.inf)
                p = (z - z.amax(-1, keepdim=True)).exp_()
                ref[r:r + 256, h] = (p_term(p).double() @ v) / p.sum(-1, keepdim=True)
        return ref


def off(x, ref):
    return float((x - ref).norm() / ref.norm())


@pytest.mark.parametrize("dtype", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("seqs,rows,ctx,heads,kvh,hd", [
    (600, 1, 20001, 1, 1, 64),      # more sequences than CTAs: a warp goes through a quarter of a context
    (600, 1, 131072, 1, 1, 64),
    (450, 1, 16380, 8, 1, 128),
    (300, 2, 8190, 6, 1, 32),       # 12 rows of a kv head
    (3, 1, 100003, 4, 2, 128),      # few sequences: split over the GPU
])
def test_long_contexts_keep_the_accuracy_of_short_ones(be, dtype, seqs, rows, ctx, heads, kvh, hd):
    s = Shared(seqs, rows, ctx, heads, kvh, hd, dtype)
    got, ref = s.attend(be), s.formula()
    own = off(ref.to(TYPES[dtype][0]).double(), ref)
    few = rows * heads // kvh <= 8
    p = 0.0 if dtype == "f32" or dtype == "f16" and few else 2.0 ** -11 / math.sqrt(3)
    assert off(got, ref) <= 1.01 * math.sqrt(own ** 2 + p ** 2 + 2.0 ** -36)


@pytest.mark.parametrize("seqs,rows,ctx,heads,kvh,hd", [
    (9, 1, 31, 8, 2, 128), (9, 1, 64, 4, 4, 64), (5, 1, 640, 32, 8, 128), (3, 1, 2500, 14, 2, 64),
    (40, 1, 5000, 8, 1, 128), (1, 1, 9000, 8, 8, 32), (3, 20, 700, 8, 2, 128), (2, 130, 3000, 14, 2, 64), (1, 513, 4000, 4, 1, 128)])
def test_f32_rows_carry_f32(be, seqs, rows, ctx, heads, kvh, hd):
    s = Shared(seqs, rows, ctx, heads, kvh, hd, "f32")
    ref = s.formula()
    assert off(s.attend(be), ref) <= 1.2e-6
    for half in (dict(q_term=lambda x: x.half()), dict(p_term=lambda x: x.half())):
        assert off(s.formula(**half), ref) > 1e-5
