"""The 8-bit paged KV cache (pox_cuda_qk_norm_rope, pox_cuda_kv8_append / _read / _attention) against plain
implementations in 64 bits.

Bounds. u is the unit roundoff of the rows' type (2^-24, 2^-11, 2^-8); sums of n f32 terms are off by at most
n 2^-24 of the sum of magnitudes.
  * q/k rows: the norm's factor carries at most (hd / 2 + 8) 2^-24, the rotation two products and a sum; against the pair's
    magnitude |a| + |b| that is (hd / 2 + 12) 2^-24, plus u of the result.
  * stored bytes: the rule is elementwise f32 arithmetic, so a numpy f32 restatement gives the same bytes; against the
    64-bit values a first store is off by half a step, and each growth of the scale adds at most half a step more.
  * attention: a score's error e_s <= (hd + 8) 2^-24 sum |q k| scale (2 for the exponent's base change) moves a
    probability by e_s; f16 and bf16 rows round p to 11 bits (2^-11); the sums of p and p v add 64 2^-24 with
    pairwise partials. Against max |v|: 2 e_s + 2^-18 (f32) or 2 e_s + 2^-10 (f16, bf16), plus u of the result.
"""
import math

import numpy as np
import pytest

from paraoxidizer_b200 import _lib as L
from paraoxidizer_b200.backend import CudaBackend

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

PAGE = 16
STREAM = 1  # the legacy default stream, on which torch works here
TYPES = {"f32": (torch.float32, L.POX_F32, 2.0 ** -24), "f16": (torch.float16, L.POX_F16, 2.0 ** -11),
         "bf16": (torch.bfloat16, L.POX_BF16, 2.0 ** -8)}


@pytest.fixture(scope="module")
def be():
    b = CudaBackend.create(0)
    yield b
    b.synchronize()
    b.close()


def rows_of(t):
    code = {torch.float32: L.POX_F32, torch.float16: L.POX_F16, torch.bfloat16: L.POX_BF16}[t.dtype]
    return L.Rows(t.data_ptr(), code, t.stride(0), t.stride(1))


def layouts(shape, dtype, kind):
    """An empty [rows][heads][hd] view: packed, a slice of longer rows, head-major, or off the vector alignment."""
    r, h, d = shape
    if kind == "packed":
        return torch.zeros(r, h, d, dtype=dtype, device="cuda")
    if kind == "fused":
        return torch.zeros(r, h + 3, d, dtype=dtype, device="cuda")[:, 2:2 + h]
    if kind == "headmajor":
        return torch.zeros(h, r, d, dtype=dtype, device="cuda").transpose(0, 1)
    big = torch.zeros(r * (h * d + 3) + 1, dtype=dtype, device="cuda")  # "odd": odd strides, odd base
    return big[1:].as_strided((r, h, d), (h * d + 3, d, 1), 1)


def rope_table(n, rot, base=10000.0):
    a = np.arange(n)[:, None] * base ** (-np.arange(0, rot, 2) / rot)
    return torch.from_numpy(np.stack([np.cos(a), np.sin(a)], -1).astype(np.float32)).cuda()


def turn64(x, table, pos, rot, half):
    """x [rows][heads][hd] (64 bits) with its first rot dims rotated by the table's rows at pos."""
    if not rot:
        return x
    c, s = table.double()[pos][:, None].unbind(-1)
    y = x.clone()
    i = torch.arange(rot // 2, device=x.device)
    lo, hi = (i, i + rot // 2) if half else (2 * i, 2 * i + 1)
    y[..., lo] = x[..., lo] * c - x[..., hi] * s
    y[..., hi] = x[..., lo] * s + x[..., hi] * c
    return y


# ---- norms and rotation ---------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("rows,heads,kvh,hd,rot,half,norm,kind", [
    (1, 32, 8, 128, 128, False, True, "fused"),
    (7, 4, 4, 64, 32, True, True, "packed"),
    (33, 5, 1, 128, 64, False, False, "headmajor"),
    (300, 14, 2, 64, 64, True, True, "odd"),
    (5, 3, 3, 96, 24, True, True, "packed"),
    (9, 2, 1, 256, 256, True, True, "packed"),
    (3, 1, 1, 34, 10, False, True, "packed"),
    (257, 0, 8, 128, 128, True, True, "fused"),
    (6, 6, 0, 32, 0, False, True, "packed"),
    (2, 1, 1, 512, 512, False, True, "packed"),
])
def test_qk_norm_rope(be, dtype, rows, heads, kvh, hd, rot, half, norm, kind):
    dt, _, u = TYPES[dtype]
    g = torch.Generator(device="cuda").manual_seed(rows * 7 + hd)
    table = rope_table(500, rot) if rot else None
    pos = torch.randint(0, 500, (rows,), generator=g, device="cuda", dtype=torch.int32)
    args, ref = L.QkNormRope(), []
    args.rows, args.heads, args.kv_heads, args.head_dim, args.eps = rows, heads, kvh, hd, 1e-5
    if rot:
        args.rope = L.Rope(table.data_ptr(), 500, rot, L.POX_ROPE_HALF if half else L.POX_ROPE_INTERLEAVED)
        args.positions = pos.data_ptr()
    for side, h in (("q", heads), ("k", kvh)):
        if not h:
            continue
        x, y = layouts((rows, h, hd), dt, kind), layouts((rows, h, hd), dt, kind)
        x.copy_(torch.randn(rows, h, hd, generator=g, device="cuda") * 3)
        w = (1 + 0.3 * torch.randn(hd, generator=g, device="cuda")).half()
        setattr(args, side, rows_of(x))
        setattr(args, side + "_out", rows_of(y))
        if norm:
            setattr(args, side + "_norm", w.data_ptr())
        z = x.double()
        if norm:
            z = z / (z.pow(2).mean(-1, keepdim=True) + 1e-5).sqrt() * w.double()
        e = turn64(z, table, pos.long(), rot, half)
        mag = z.abs()
        if rot:
            i = torch.arange(rot // 2, device="cuda")
            lo, hi = (i, i + rot // 2) if half else (2 * i, 2 * i + 1)
            both = mag[..., lo] + mag[..., hi]
            mag[..., lo] = both
            mag[..., hi] = both
        ref.append((x, y, w, e, mag))
    be.qk_norm_rope(args, STREAM)
    be.synchronize()
    for x, y, w, e, mag in ref:
        tol = (hd / 2 + 12) * 2.0 ** -24 * mag + u * e.abs() * 1.01 + 2.0 ** -25 * (dtype == "f16")
        assert bool(((y.double() - e).abs() <= tol).all())
    # in place
    for side, h in (("q", heads), ("k", kvh)):
        if h:
            setattr(args, side + "_out", getattr(args, side))
    be.qk_norm_rope(args, STREAM)
    be.synchronize()
    for x, y, *_ in ref:
        assert torch.equal(x, y)


def test_qk_norm_rope_position_outside_the_table(be):
    x = torch.ones(3, 2, 64, device="cuda")
    y = torch.full_like(x, 7.0)
    table, pos = rope_table(8, 64), torch.tensor([2, 8, 3], dtype=torch.int32, device="cuda")
    a = L.QkNormRope(rows_of(x), L.Rows(), rows_of(y), L.Rows(), 3, 2, 0, 64, 0, 0, 1e-5,
                     L.Rope(table.data_ptr(), 8, 64, L.POX_ROPE_HALF), pos.data_ptr())
    be.qk_norm_rope(a, STREAM)
    with pytest.raises(L.PoxError, match="rotation table"):
        be.synchronize()
    assert bool((y[1] == 7).all()) and not bool((y[0] == 7).any()) and not bool((y[2] == 7).any())


# ---- the cache -------------------------------------------------------------------------------------------------
class Cache:
    """Pages, scales and block tables of sequences with room for `ctx` tokens each, pages scattered."""

    def __init__(self, ctx, kvh, hd, seed=0, fill=True, spread=0.6):
        rng = np.random.default_rng(seed)
        self.kvh, self.hd, self.width = kvh, hd, max(1, max((c + PAGE - 1) // PAGE for c in ctx)) + 1
        need = [(c + PAGE - 1) // PAGE for c in ctx]
        self.blocks = sum(need) + 2
        perm = rng.permutation(self.blocks)
        tab = np.full((len(ctx), self.width), -1, np.int32)
        o = 0
        for i, n in enumerate(need):
            tab[i, :n] = perm[o:o + n]
            o += n
        self.tab_np, self.tab = tab, torch.from_numpy(tab).cuda()
        g = torch.Generator(device="cuda").manual_seed(seed)
        self.pages = torch.zeros(self.blocks, kvh, 32 * hd, dtype=torch.int8, device="cuda")
        self.scales = torch.full((self.blocks, kvh, 2), float("nan"), device="cuda")
        if fill:
            self.pages.copy_((torch.randn(self.pages.shape, generator=g, device="cuda") * 36).round().clamp(-127, 127))
            self.scales.copy_(torch.rand(self.scales.shape, generator=g, device="cuda").mul(spread).exp() * 0.02)
        self.c = L.Kv8Cache(self.pages.data_ptr(), self.scales.data_ptr(), self.blocks, kvh, hd)

    def batch(self, starts, ctx):
        self.keep = getattr(self, "keep", [])
        n = [b - a for a, b in zip(starts, starts[1:])]
        st = torch.tensor(starts, dtype=torch.int32, device="cuda")
        cx = torch.tensor(ctx, dtype=torch.int32, device="cuda")
        self.keep += [st, cx]
        one = all(x == 1 for x in n)
        return L.Kv8Batch(0 if one else st.data_ptr(), cx.data_ptr(), self.tab.data_ptr(), len(ctx), starts[-1], max(n),
                          max(max(ctx), 1), self.width)

    def values(self, s, ctx, side):
        """[ctx][kv head][hd] in 64 bits: what the pages of sequence s hold (0: k, 1: v), by the documented layout."""
        hd, nb = self.hd, (ctx + PAGE - 1) // PAGE
        ids = torch.from_numpy(self.tab_np[s, :nb].astype(np.int64)).cuda()
        t, d = torch.meshgrid(torch.arange(PAGE), torch.arange(hd), indexing="ij")
        at = 16 * hd + 16 * d + t if side else t * hd + (d ^ (64 * (t % 2)) if hd == 128 else d)
        x = self.pages[ids][..., at.cuda()].double() * self.scales[ids][..., side, None, None].double()
        return x.permute(0, 2, 1, 3).reshape(nb * PAGE, self.kvh, hd)[:ctx]


def np_append(pages, scales, c, tab, starts, ctx, k, v, table, rot, half):
    """The append's rule in numpy f32, page by page (pages / scales: numpy copies, updated)."""
    f = np.float32
    hd = c.hd
    for s, (a, b) in enumerate(zip(starts, starts[1:])):
        p0 = max(ctx[s] - (b - a), 0)
        for page in range(p0 // PAGE, (ctx[s] + PAGE - 1) // PAGE):
            blk, first, last = tab[s, page], max(p0 - page * PAGE, 0), min(ctx[s] - page * PAGE, PAGE)
            pos = np.arange(page * PAGE + first, page * PAGE + last)
            if not len(pos):  # a sequence without rows in this call
                continue
            r = a + pos - (ctx[s] - (b - a))
            for side, src in ((0, k), (1, v)):
                x = src[r].astype(f)
                if side == 0 and rot:
                    cs = table[pos][:, None]
                    i = np.arange(rot // 2)
                    lo, hi = (i, i + rot // 2) if half else (2 * i, 2 * i + 1)
                    y = x.copy()
                    y[..., lo] = x[..., lo] * cs[..., 0] - x[..., hi] * cs[..., 1]
                    y[..., hi] = x[..., lo] * cs[..., 1] + x[..., hi] * cs[..., 0]
                    x = y
                fin = np.where(np.isfinite(x), np.abs(x), f(0))
                m = fin.max((0, 2))
                old = scales[blk, :, side] if first else np.zeros(c.kvh, f)
                now = np.maximum(old, m / f(127))
                ratio = np.where(now > 0, old / np.where(now > 0, now, 1), f(0)).astype(f)
                t, d = np.meshgrid(np.arange(PAGE), np.arange(hd), indexing="ij")
                at = 16 * hd + 16 * d + t if side else t * hd + (d ^ (64 * (t % 2)) if hd == 128 else d)
                for h in range(c.kvh):
                    pg = pages[blk, h]
                    pg[at[:first]] = np.rint(pg[at[:first]].astype(f) * ratio[h]).astype(np.int8)
                    q = x[:, h] / now[h] if now[h] > 0 else np.zeros_like(x[:, h])
                    q = np.where(np.isnan(q), 0, np.clip(np.rint(q), -127, 127))
                    pg[at[first:last]] = q.astype(np.int8)
                scales[blk, :, side] = now


CHUNKS = [
    ([0, 1], [1]),                                  # the first token of a sequence
    ([0, 16], [16]),                                # one whole page
    ([0, 17, 18, 18, 50], [17, 33, 40, 47]),        # a page and one more; one row; no row; a chunk from slot 15
    ([0, 1, 2, 3, 4], [1, 16, 17, 700]),            # decode: slots 0, 15, 0, 11
    ([0, 1, 3, 4], [0, 1, 5]),                      # padding: a free slot, two rows of which one is padding
    ([0, 301, 812], [333, 511]),                    # long chunks, from inside a page and from the start
]


@pytest.mark.parametrize("starts,ctx", CHUNKS)
@pytest.mark.parametrize("dtype,hd,kvh,rot,half,kind", [
    ("f32", 128, 2, 128, False, "packed"), ("bf16", 128, 8, 128, True, "fused"), ("f16", 64, 3, 32, True, "headmajor"),
    ("f16", 32, 1, 0, False, "odd"), ("f32", 64, 5, 24, True, "odd"), ("bf16", 32, 4, 32, False, "packed"),
    ("f32", 128, 1, 6, True, "fused")])
def test_append_stores_the_rule_and_read_returns_it(be, starts, ctx, dtype, hd, kvh, rot, half, kind):
    dt = TYPES[dtype][0]
    c = Cache([max(x, 1) for x in ctx], kvh, hd, seed=sum(ctx))
    g = torch.Generator(device="cuda").manual_seed(hd + starts[-1])
    k, v = (layouts((starts[-1], kvh, hd), dt, kind) for _ in range(2))
    k.copy_(torch.randn(k.shape, generator=g, device="cuda") * 2)
    v.copy_(torch.randn(v.shape, generator=g, device="cuda"))
    table = rope_table(max(ctx) + 1, rot) if rot else None
    rope = L.Rope(table.data_ptr(), max(ctx) + 1, rot, L.POX_ROPE_HALF if half else 0) if rot else None
    pages, scales = c.pages.cpu().numpy(), c.scales.cpu().numpy()
    np_append(pages, scales, c, c.tab_np, starts, ctx, k.float().cpu().numpy(), v.float().cpu().numpy(),
              table.cpu().numpy() if rot else None, rot, half)
    batch = c.batch(starts, ctx)
    be.kv8_append(c.c, batch, rows_of(k), rows_of(v), rope, STREAM)
    be.synchronize()
    assert np.array_equal(c.scales.cpu().numpy(), scales)
    assert np.array_equal(c.pages.cpu().numpy(), pages)
    ko, vo = (layouts((starts[-1], kvh, hd), dt, kind) for _ in range(2))
    be.kv8_read(c.c, batch, rows_of(ko), rows_of(vo), STREAM)
    be.synchronize()
    for s, (a, b) in enumerate(zip(starts, starts[1:])):
        n = min(b - a, ctx[s])
        assert not bool(ko[a:b - n].any()) and not bool(vo[a:b - n].any())
        if not n:
            continue
        pos = torch.arange(ctx[s] - n, ctx[s], device="cuda")
        exact = turn64(k[b - n:b].double(), table, pos, rot, half), v[b - n:b].double()
        for side, got in enumerate((ko, vo)):
            held = c.values(s, ctx[s], side)[ctx[s] - n:]
            assert torch.equal(got[b - n:b], held.float().to(dt)) or bool(
                ((got[b - n:b].double() - held).abs() <= TYPES[dtype][2] * held.abs() + 2.0 ** -25).all())
            ids = torch.from_numpy(c.tab_np[s].astype(np.int64)).cuda()[pos // PAGE]
            step = c.scales[ids][..., side, None].double()
            assert bool(((held - exact[side]).abs() <= step * (0.5 + 2.0 ** -10)).all())


def test_append_token_by_token_stays_within_its_steps(be):
    """Growing magnitudes: every token raises the scale of its page. The error of an element is at most half a step for
    its store and for each later growth, in steps of the scale at that time (all at most the last one)."""
    kvh, hd, n = 2, 64, 37
    c = Cache([n], kvh, hd, fill=False)
    g = torch.Generator(device="cuda").manual_seed(5)
    x = torch.randn(n, kvh, hd, generator=g, device="cuda") * (1 + torch.arange(n, device="cuda")[:, None, None] * 0.1)
    for i in range(n):
        be.kv8_append(c.c, c.batch([0, 1], [i + 1]), rows_of(x[i:i + 1]), rows_of(x[i:i + 1] * 3), None, STREAM)
    be.synchronize()
    for side, f in ((0, 1.0), (1, 3.0)):
        held = c.values(0, n, side)
        step = c.scales[c.tab[0, :(n + 15) // 16].long()][..., side].double().repeat_interleave(PAGE, 0)[:n, :, None]
        later = torch.tensor([min((i // PAGE + 1) * PAGE, n) - i for i in range(n)], device="cuda")[:, None, None]
        assert bool(((held - x.double() * f).abs() <= step * (0.5 * later + 0.01)).all())
        most = (x.double() * f).abs().amax(2)  # the scale is that of the largest element, to an ulp
        for p in range(0, n, PAGE):
            assert torch.allclose(step[p, :, 0] * 127, most[p:p + PAGE].amax(0), rtol=2.0 ** -22)


def test_append_of_elements_that_are_not_finite(be):
    c = Cache([16], 1, 64, fill=False)
    x = torch.zeros(3, 1, 64, device="cuda")
    x[0, 0, :4] = torch.tensor([1.0, float("inf"), float("-inf"), float("nan")])
    x[1, 0, 0] = -2.54
    v = torch.full_like(x, float("nan"))
    be.kv8_append(c.c, c.batch([0, 3], [3]), rows_of(x), rows_of(v), None, STREAM)
    ko, vo = torch.empty_like(x), torch.empty_like(x)
    be.kv8_read(c.c, c.batch([0, 3], [3]), rows_of(ko), rows_of(vo), STREAM)
    be.synchronize()
    s = 2.54 / 127
    assert torch.allclose(ko[0, 0, :4], torch.tensor([50 * s, 127 * s, -127 * s, 0.0], device="cuda"), rtol=1e-6)
    assert torch.allclose(ko[1, 0, 0], torch.tensor(-2.54, device="cuda"), rtol=1e-6)
    assert not bool(vo.any()) and not bool(ko[2].any())  # a page of nothing holds zeros


# ---- attention -------------------------------------------------------------------------------------------------
def attend64(c, starts, ctx, q, scale):
    """(out, max |v|, largest score error's factor) in 64 bits, sequence by sequence."""
    rows, heads, hd = q.shape
    group = heads // c.kvh
    out = torch.zeros(rows, heads, hd, dtype=torch.float64, device="cuda")
    tol = torch.zeros(rows, heads, 1, dtype=torch.float64, device="cuda")
    for s, (a, b) in enumerate(zip(starts, starts[1:])):
        if b == a or ctx[s] == 0:
            continue
        k, v = c.values(s, ctx[s], 0), c.values(s, ctx[s], 1)
        last = torch.arange(ctx[s] - (b - a), ctx[s], device="cuda")
        seen = torch.arange(ctx[s], device="cuda")[None] <= last[:, None]
        for h in range(heads):
            kh, vh, qh = k[:, h // group], v[:, h // group], q[a:b, h].double()
            z = (qh @ kh.T * scale).masked_fill(~seen, -math.inf)
            p = torch.nan_to_num(torch.softmax(z, -1), nan=0.0)
            out[a:b, h] = torch.where(seen, p, torch.zeros_like(p)) @ vh
            mag = (qh.abs() @ kh.abs().T * scale).masked_fill(~seen, 0).amax(1)
            vmax = (seen * vh.abs().amax(1)).amax(1)
            tol[a:b, h, 0] = vmax * 2 * (hd + 8) * 2.0 ** -24 * 2 * mag
            tol[a:b, h, 0] += vmax * (2.0 ** -18 if q.dtype == torch.float32 else 2.0 ** -10)
    return out, tol


def check_attention(be, c, starts, ctx, heads, dtype, kind="packed", scale=0.0, gain=1.0, seed=1):
    dt, _, u = TYPES[dtype]
    g = torch.Generator(device="cuda").manual_seed(seed)
    q, out = (layouts((starts[-1], heads, c.hd), dt, kind) for _ in range(2))
    q.copy_(torch.randn(q.shape, generator=g, device="cuda") * gain)
    out.fill_(float("nan"))
    be.kv8_attention(c.c, c.batch(starts, ctx), rows_of(q), rows_of(out), heads, scale, STREAM)
    be.synchronize()
    ref, tol = attend64(c, starts, ctx, q, scale or 1 / math.sqrt(c.hd))
    err = (out.double() - ref).abs()
    bad = ~(err <= tol + u * 1.01 * ref.abs() + 2.0 ** -25 * (dtype == "f16"))
    assert not bool(bad.any()), (int(bad.sum()), float(err.nan_to_num(nan=1e9).max()), bad.nonzero()[:4].tolist())
    again = torch.empty_like(out)
    again = again.as_strided(out.shape, again.stride())
    be.kv8_attention(c.c, c.batch(starts, ctx), rows_of(q), rows_of(again), heads, scale, STREAM)
    be.synchronize()
    assert torch.equal(out, again)  # the same call gives the same bits


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("heads,kvh,hd,kind", [(4, 4, 64, "packed"), (32, 8, 128, "fused"), (8, 1, 128, "headmajor"),
                                               (14, 2, 64, "odd"), (5, 1, 32, "packed"), (32, 2, 64, "packed"),
                                               (24, 1, 128, "odd")])
def test_attention_of_single_tokens(be, dtype, heads, kvh, hd, kind):
    ctx = [1, 0, 15, 16, 17, 31, 64, 65, 129, 640, 1023, 2500]
    c = Cache(ctx, kvh, hd, seed=heads)
    check_attention(be, c, list(range(len(ctx) + 1)), ctx, heads, dtype, kind)


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("heads,kvh,hd", [(8, 2, 128), (7, 1, 64), (3, 3, 64), (4, 2, 32), (40, 2, 128)])
def test_attention_of_ragged_chunks(be, dtype, heads, kvh, hd):
    n = [1, 3, 0, 17, 130, 2, 64, 1, 300]
    ctx = [0, 3, 0, 40, 130, 1, 700, 333, 1111]  # a free slot, a whole prompt, no row, ..., one of two rows is padding
    starts = np.concatenate([[0], np.cumsum(n)]).tolist()
    c = Cache(ctx, kvh, hd, seed=3)
    check_attention(be, c, starts, ctx, heads, dtype)


@pytest.mark.parametrize("dtype,rows", [("bf16", 1000), ("f16", 1025), ("f32", 513)])
@pytest.mark.parametrize("hd", [64, 128])
def test_attention_of_a_prompt(be, dtype, rows, hd):
    c = Cache([rows + 37], 2, hd, seed=9)
    check_attention(be, c, [0, rows], [rows + 37], 8, dtype)


def test_attention_over_a_long_context(be):
    c = Cache([30001, 70], 2, 128, seed=4)
    check_attention(be, c, [0, 1, 2], [30001, 70], 8, "f16")
    check_attention(be, c, [0, 2, 5], [30001, 70], 8, "f32")


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("n", [1, 40])
def test_attention_scores_far_apart_and_scales_far_apart(be, dtype, n):
    """Large queries put all the weight on one token; pages whose scales differ by 10^6; a page whose scale is zero."""
    ctx = [200, 333]
    starts = [0, n, 2 * n]
    c = Cache(ctx, 2, 128, seed=11)
    check_attention(be, c, starts, ctx, 8, dtype, gain=30.0)
    c.scales[c.tab[0, 3].item(), :, 1] *= 1e6
    c.scales[c.tab[0, 5].item(), :, 1] *= 1e-6
    c.scales[c.tab[1, 2].item(), :, :] = 0.0
    check_attention(be, c, starts, ctx, 8, dtype)
    check_attention(be, c, starts, ctx, 8, dtype, scale=0.01)


def test_attention_ignores_what_no_row_sees(be):
    """NaN and infinite scales in pages past the context, and in a page that only later rows of the chunk see."""
    c = Cache([100, 100], 1, 64, seed=2)
    ref = torch.empty(60, 4, 64, device="cuda")
    q = torch.randn(60, 4, 64, device="cuda")
    b = c.batch([0, 30, 60], [50, 50])
    be.kv8_attention(c.c, b, rows_of(q), rows_of(ref), 4, 0.0, STREAM)
    be.synchronize()
    c.scales[c.tab[0, 4:6].long()] = float("nan")  # tokens 64 .. 95: past the context
    c.scales[c.tab[1, 3].item()] = float("inf")    # tokens 48, 49: seen by the chunk's last two rows only
    out = torch.empty_like(ref)
    be.kv8_attention(c.c, b, rows_of(q), rows_of(out), 4, 0.0, STREAM)
    be.synchronize()
    assert torch.equal(out[:58], ref[:58]) and bool(torch.isfinite(ref).all())
    assert not bool(torch.isfinite(out[58:]).all())


def test_attention_of_queries_that_are_not_finite(be):
    c = Cache([50], 1, 64, seed=2)
    q = torch.randn(3, 2, 64, device="cuda")
    q[0, 1, 5] = float("nan")
    q[2, 0, 7] = float("inf")
    out = torch.empty_like(q)
    be.kv8_attention(c.c, c.batch([0, 3], [50]), rows_of(q), rows_of(out), 2, 0.0, STREAM)
    be.synchronize()
    assert bool(torch.isnan(out[0, 1]).all()) and bool(torch.isnan(out[2, 0]).all())
    for r, h in ((0, 0), (1, 0), (1, 1), (2, 1)):
        assert bool(torch.isfinite(out[r, h]).all())


def test_on_another_stream_and_in_a_graph(be):
    """The step on a stream of its own, captured and replayed: the same bytes and outputs as eager calls."""
    kvh, hd, heads, ctx = 2, 128, 8, [33, 200, 1]
    table = rope_table(300, hd)
    rope = L.Rope(table.data_ptr(), 300, hd, L.POX_ROPE_HALF)
    x = torch.randn(3, heads + 2 * kvh, hd, device="cuda", dtype=torch.bfloat16)
    q, k, v = x[:, :heads], x[:, heads:heads + kvh], x[:, heads + kvh:]
    pos = torch.tensor([c - 1 for c in ctx], dtype=torch.int32, device="cuda")
    got = []
    for graph in (False, True):
        c = Cache(ctx, kvh, hd, seed=8)
        b, st = c.batch([0, 1, 2, 3], ctx), torch.cuda.Stream()
        qo, out = torch.empty_like(q), torch.empty(3, heads, hd, device="cuda", dtype=torch.bfloat16)
        a = L.QkNormRope(rows_of(q), L.Rows(), rows_of(qo), L.Rows(), 3, heads, 0, hd, 0, 0, 1e-5, rope, pos.data_ptr())

        def step(stream):
            be.qk_norm_rope(a, stream)
            be.kv8_append(c.c, b, rows_of(k), rows_of(v), rope, stream)
            be.kv8_attention(c.c, b, rows_of(qo), rows_of(out), heads, 0.0, stream)

        torch.cuda.synchronize()
        step(st.cuda_stream)
        torch.cuda.synchronize()
        if graph:
            out.zero_()
            gr = torch.cuda.CUDAGraph()
            with torch.cuda.graph(gr, stream=st):
                step(st.cuda_stream)
            gr.replay()
            gr.replay()
        torch.cuda.synchronize()
        got.append((out, c.pages, c.scales))
    assert all(torch.equal(i.nan_to_num(), j.nan_to_num()) for i, j in zip(*got))


# ---- refusals --------------------------------------------------------------------------------------------------
def test_refusals(be):
    c = Cache([40, 40], 2, 64)
    q, kv = torch.zeros(2, 4, 64, device="cuda"), torch.zeros(2, 2, 64, device="cuda")
    b = c.batch([0, 1, 2], [40, 40])
    call = {"append": lambda cache=c.c, batch=b, k=rows_of(kv), v=rows_of(kv), rope=None:
            be.kv8_append(cache, batch, k, v, rope, STREAM),
            "read": lambda cache=c.c, batch=b, k=rows_of(kv), v=rows_of(kv): be.kv8_read(cache, batch, k, v, STREAM),
            "attend": lambda cache=c.c, batch=b, q=rows_of(q), out=rows_of(torch.empty_like(q)), heads=4, scale=0.0:
            be.kv8_attention(cache, batch, q, out, heads, scale, STREAM)}
    for f in call.values():
        f()
    be.synchronize()

    def refused(code, name, **kw):
        with pytest.raises(L.PoxError) as e:
            call[name](**kw)
        assert e.value.code == code, (name, kw, str(e.value))

    def changed(s, **kw):
        t = type(s).from_buffer_copy(s)
        for n, v in kw.items():
            setattr(t, n, v)
        return t

    for name in call:
        refused(L.POX_ERR_INVALID, name, cache=changed(c.c, pages=None))
        refused(L.POX_ERR_INVALID, name, cache=changed(c.c, pages=c.c.pages + 4))
        refused(L.POX_ERR_INVALID, name, cache=changed(c.c, scales=c.c.scales + 4))
        refused(L.POX_ERR_UNSUPPORTED, name, cache=changed(c.c, head_dim=96))
        refused(L.POX_ERR_INVALID, name, cache=changed(c.c, kv_heads=0))
        refused(L.POX_ERR_INVALID, name, batch=changed(b, ctx_lens=None))
        refused(L.POX_ERR_INVALID, name, batch=changed(b, block_tables=b.block_tables + 2))
        refused(L.POX_ERR_INVALID, name, batch=changed(b, rows=3))
        refused(L.POX_ERR_INVALID, name, batch=changed(b, max_ctx=16 * b.max_blocks_per_seq + 1))
        call[name](batch=changed(b, rows=0, seqs=0))  # nothing to do
    for name, arg, t in (("append", "k", kv), ("read", "v", kv), ("attend", "q", q), ("attend", "out", q)):
        refused(L.POX_ERR_INVALID, name, **{arg: changed(rows_of(t), data=None)})
        refused(L.POX_ERR_INVALID, name, **{arg: changed(rows_of(t), data=t.data_ptr() + 2)})
        refused(L.POX_ERR_UNSUPPORTED, name, **{arg: changed(rows_of(t), dtype=L.POX_I8)})
        refused(L.POX_ERR_INVALID, name, **{arg: changed(rows_of(t), row_stride=2 ** 60)})
    refused(L.POX_ERR_INVALID, "append", v=rows_of(kv.half()))
    refused(L.POX_ERR_INVALID, "read", k=changed(rows_of(kv), row_stride=64))   # rows of an output overlap
    refused(L.POX_ERR_INVALID, "attend", out=changed(rows_of(q), head_stride=32))
    refused(L.POX_ERR_INVALID, "attend", heads=3)
    refused(L.POX_ERR_INVALID, "attend", heads=0)
    refused(L.POX_ERR_INVALID, "attend", scale=float("nan"))
    refused(L.POX_ERR_INVALID, "attend", scale=-1.0)
    table = rope_table(64, 64)
    refused(L.POX_ERR_INVALID, "append", rope=L.Rope(table.data_ptr(), 64, 63, 0))
    refused(L.POX_ERR_INVALID, "append", rope=L.Rope(table.data_ptr(), 64, 66, 0))
    refused(L.POX_ERR_INVALID, "append", rope=L.Rope(None, 64, 64, 0))
    refused(L.POX_ERR_UNSUPPORTED, "append", rope=L.Rope(table.data_ptr(), 64, 64, 2))

    def qk(**kw):
        a = L.QkNormRope(rows_of(q), rows_of(kv), rows_of(q), rows_of(kv), 2, 4, 2, 64, 0, 0, 1e-5, L.Rope(), 0)
        be.qk_norm_rope(changed(a, **kw), STREAM)

    qk()
    for code, kw in ((L.POX_ERR_UNSUPPORTED, dict(head_dim=63)), (L.POX_ERR_UNSUPPORTED, dict(head_dim=514)),
                     (L.POX_ERR_INVALID, dict(k=rows_of(kv.half()), k_out=rows_of(kv.half()))),
                     (L.POX_ERR_INVALID, dict(q_out=changed(rows_of(q), head_stride=32))),
                     (L.POX_ERR_INVALID, dict(q=changed(rows_of(q), head_stride=128))),
                     (L.POX_ERR_INVALID, dict(rope=L.Rope(table.data_ptr(), 64, 64, 0))),
                     (L.POX_ERR_INVALID, dict(q=L.Rows()))):
        with pytest.raises(L.PoxError) as e:
            qk(**kw)
        assert e.value.code == code, (kw, str(e.value))
    be.synchronize()


def test_bad_input_on_the_device_is_left_out_and_reported(be):
    c = Cache([40, 40], 1, 64, seed=1)
    q = torch.randn(2, 2, 64, device="cuda")
    out = torch.zeros_like(q)
    good = torch.zeros_like(q)
    b = c.batch([0, 1, 2], [40, 40])
    be.kv8_attention(c.c, b, rows_of(q), rows_of(good), 2, 0.0, STREAM)
    be.synchronize()
    for page in (-1, c.blocks, 2 ** 31 - 1):
        c.tab[0, 1] = page
        be.kv8_attention(c.c, b, rows_of(q), rows_of(out), 2, 0.0, STREAM)
        with pytest.raises(L.PoxError, match="block-table entry"):
            be.synchronize()
        assert torch.equal(out[1], good[1]) and bool(torch.isfinite(out).all())
        kv = torch.randn(2, 1, 64, device="cuda")
        before = c.pages.clone()
        be.kv8_append(c.c, c.batch([0, 1, 2], [20, 0]), rows_of(kv), rows_of(kv), None, STREAM)
        with pytest.raises(L.PoxError, match="block-table entry"):
            be.synchronize()
        assert torch.equal(before, c.pages)
    # a sequence longer than the batch says, row starts past the rows: that sequence is left out
    short = L.Kv8Batch.from_buffer_copy(b)
    short.max_ctx = 39
    out.fill_(5.0)
    be.kv8_attention(c.c, short, rows_of(q), rows_of(out), 2, 0.0, STREAM)
    with pytest.raises(L.PoxError, match="bounds"):
        be.synchronize()
    assert bool((out == 5.0).all())


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_row_starts_that_descend_are_reported(be, dtype):
    """A sequence of fewer than no rows owns no work, and is reported all the same; the others are computed."""
    dt = TYPES[dtype][0]
    ctx = [300, 300, 300]
    c = Cache(ctx, 1, 64, seed=3)
    b = c.batch([0, 300, 150, 450], ctx)
    b.max_rows = 300
    q, out = (torch.randn(450, 4, 64, device="cuda").to(dt) for _ in range(2))
    kv = torch.randn(450, 1, 64, device="cuda").to(dt)
    for call in (lambda: be.kv8_append(c.c, b, rows_of(kv), rows_of(kv), None, STREAM),
                 lambda: be.kv8_read(c.c, b, rows_of(kv), rows_of(kv.clone()), STREAM),
                 lambda: be.kv8_attention(c.c, b, rows_of(q), rows_of(out), 4, 0.0, STREAM)):
        call()
        with pytest.raises(L.PoxError, match="bounds"):
            be.synchronize()
    assert bool(torch.isfinite(out).all())


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_attention_of_a_prompt_among_single_tokens(be, dtype):
    """One prompt among many decoding sequences, with a bound of the rows that says nothing."""
    n = [1] * 21 + [700] + [1] * 33 + [0, 300]
    ctx = [1 + 7 * i for i in range(21)] + [900] + [16 * i + 1 for i in range(33)] + [5, 300]
    starts = [0]
    for i in n:
        starts.append(starts[-1] + i)
    c = Cache(ctx, 2, 128, seed=4)
    batch = c.batch

    def loose(*a):
        b = batch(*a)
        b.max_rows = 2 ** 31
        return b

    c.batch = loose
    check_attention(be, c, starts, ctx, 8, dtype)


def test_a_graph_outlives_larger_calls_on_its_stream(be):
    st = torch.cuda.Stream()
    small, ctx = Cache([900], 2, 64, seed=5), [100 + 31 * i for i in range(70)]
    large = Cache(ctx, 4, 128, seed=6)
    bs, bl = small.batch([0, 1], [900]), large.batch(list(range(71)), ctx)
    q, out = torch.randn(1, 4, 64, device="cuda"), torch.empty(1, 4, 64, device="cuda")
    ql, outl = (torch.randn(70, 64, 128, device="cuda") for _ in range(2))
    torch.cuda.synchronize()
    be.kv8_attention(small.c, bs, rows_of(q), rows_of(out), 4, 0.0, st.cuda_stream)
    torch.cuda.synchronize()
    want = out.clone()
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr, stream=st):
        be.kv8_attention(small.c, bs, rows_of(q), rows_of(out), 4, 0.0, st.cuda_stream)
    be.kv8_attention(large.c, bl, rows_of(ql), rows_of(outl), 64, 0.0, st.cuda_stream)
    torch.cuda.synchronize()
    out.zero_()
    with torch.cuda.stream(st):
        gr.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, want)


def test_attention_refuses_more_rows_than_it_counts(be):
    c = Cache([16], 1, 64, seed=7)
    q = torch.zeros(1, 128, 64, device="cuda")
    b = c.batch([0, 1], [16])
    b.row_starts, b.rows, b.max_rows = c.keep[0].data_ptr(), 2 ** 24, 2 ** 24
    with pytest.raises(L.PoxError) as e:
        be.kv8_attention(c.c, b, rows_of(q), rows_of(torch.empty_like(q)), 128, 0.0, STREAM)
    assert e.value.code == L.POX_ERR_UNSUPPORTED
