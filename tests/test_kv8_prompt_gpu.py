"""Attention of prompts over the 8-bit cache by the tensor-memory kernel (f16 and bf16, head dims 64 and 128).

Which kernel a batch takes is a rule on sizes, restated here (`route`); each case says which one it is for, so that a
change of the rule shows up as a case that no longer tests what it names.

Bounds, against the formula in 64 bits. p is rounded to 11 bits: at most 2^-11 of itself, and 2^-25 of the largest where
it is subnormal in f16; a score's error e (hd products of q and k in f32, and the exponent's base) moves p by e. So an
element is off by at most (2^-11 + 2 e + 2^-16) sum p |v| + n 2^-25 max |v|, plus the rounding to the rows' type. In
norm, over independent values, the rounding of p is 2^-11 / sqrt(3) of the outputs (root mean square)."""
import math

import pytest
from test_kv8_gpu import STREAM, TYPES, Cache, layouts, rows_of

from paraoxidizer_b200 import _lib as L
from paraoxidizer_b200.backend import CudaBackend

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


@pytest.fixture(scope="module")
def be():
    b = CudaBackend.create(0)
    yield b
    b.synchronize()
    b.close()


def route(starts, max_rows, max_ctx, heads, kvh, hd, dtype):
    """"step", "prompt" or "both": what pox_cuda_kv8_attention launches."""
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    seqs, rows, group = len(starts) - 1, starts[-1], heads // kvh
    most, wide = min(max_rows, rows) * group, hd == 128
    if hd == 32 or dtype == "f32" or most <= 64:
        return "step"
    step = kvh * (rows * group / 16 + seqs / 2) * (max_ctx / 16) * (0.65 if wide else 0.46)
    ctas = kvh * (rows * group / 256 + seqs / 2)
    tile = (2350 if wide else 2050) if most <= 128 else (2750 if wide else 2350)
    if max(1.0, ctas / sms) * (max_ctx / 128) * tile >= step:
        return "step"
    return "both" if seqs > 1 and rows != seqs * max_rows else "prompt"


def formula(c, starts, ctx, q, scale, without=()):
    """(outputs, sum p |v|, max |v|, the largest sum of |q k| scale of a row) in 64 bits; `without`: pages (sequence,
    page) that are left out."""
    rows, heads, hd = q.shape
    group = heads // c.kvh
    out, mag = (torch.zeros(rows, heads, hd, dtype=torch.float64, device="cuda") for _ in range(2))
    vmax, e = (torch.zeros(rows, heads, 1, dtype=torch.float64, device="cuda") for _ in range(2))
    for s, (a, b) in enumerate(zip(starts, starts[1:])):
        if b == a or ctx[s] == 0:
            continue
        k, v = c.values(s, ctx[s], 0), c.values(s, ctx[s], 1)
        t = torch.arange(ctx[s], device="cuda")
        seen = t[None] <= torch.arange(ctx[s] - (b - a), ctx[s], device="cuda")[:, None]
        for w, page in without:
            if w == s:
                seen = seen & (t // 16 != page)
        for h in range(heads):
            kh, vh, qh = k[:, h // group].nan_to_num(0, 0, 0), v[:, h // group].nan_to_num(0, 0, 0), q[a:b, h].double()
            z = (qh @ kh.T * scale).masked_fill(~seen, -math.inf)
            p = torch.softmax(z, -1).nan_to_num(0)
            out[a:b, h], mag[a:b, h] = p @ vh, p @ vh.abs()
            vmax[a:b, h, 0] = (seen * vh.abs().amax(1)).amax(1)
            e[a:b, h, 0] = (qh.abs() @ kh.abs().T * scale).masked_fill(~seen, 0).amax(1)
    return out, mag, vmax, e * (hd + 8) * 2.0 ** -24


def run(be, c, starts, ctx, q, out, heads, kernel, dtype, scale=0.0):
    b = c.batch(starts, ctx)
    assert route(starts, b.max_rows, b.max_ctx, heads, c.kvh, c.hd, dtype) == kernel
    out.fill_(float("nan"))
    be.kv8_attention(c.c, b, rows_of(q), rows_of(out), heads, scale, STREAM)


def check(be, c, starts, ctx, heads, dtype, kernel, kind="packed", scale=0.0, gain=1.0, seed=1, norm=True):
    dt, _, u = TYPES[dtype]
    g = torch.Generator(device="cuda").manual_seed(seed)
    q, out = (layouts((starts[-1], heads, c.hd), dt, kind) for _ in range(2))
    q.copy_(torch.randn(q.shape, generator=g, device="cuda") * gain)
    run(be, c, starts, ctx, q, out, heads, kernel, dtype, scale)
    be.synchronize()
    ref, mag, vmax, e = formula(c, starts, ctx, q, scale or 1 / math.sqrt(c.hd))
    err, own = (out.double() - ref).abs(), (ref.to(dt).double() - ref).norm() / ref.norm()
    tol = (2.0 ** -11 + 2 * e + 2.0 ** -16) * mag + max(ctx) * 2.0 ** -25 * vmax
    tol += 1.01 * u * ref.abs() + 2.0 ** -25 * (dtype == "f16")
    over = torch.isinf(out) & (out.sign() == ref.sign()) & (ref.abs() + tol >= torch.finfo(dt).max)  # f16 holds 65504
    bad = ~(err <= tol) & ~over
    assert not bool(bad.any()), (int(bad.sum()), float(err.nan_to_num(nan=1e9).max()), bad.nonzero()[:4].tolist())
    if norm:
        assert float(err.norm() / ref.norm()) <= 1.01 * math.sqrt(float(own) ** 2 + 2.0 ** -22 / 3 + 2.0 ** -32)
    again = layouts((starts[-1], heads, c.hd), dt, kind)
    run(be, c, starts, ctx, q, again, heads, kernel, dtype, scale)
    be.synchronize()
    assert torch.equal(out, again)  # the same call gives the same bits


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("rows,prefix,heads,kvh,kind", [
    (1000, 0, 32, 8, "packed"), (1025, 37, 32, 8, "odd"), (511, 500, 28, 4, "fused"), (769, 3, 16, 16, "headmajor"),
    (2049, 0, 14, 2, "odd")])
def test_one_prompt(be, dtype, hd, rows, prefix, heads, kvh, kind):
    c = Cache([rows + prefix], kvh, hd, seed=rows)
    check(be, c, [0, rows], [rows + prefix], heads, dtype, "prompt", kind)


@pytest.mark.parametrize("dtype,hd", [("f16", 64), ("bf16", 128)])
@pytest.mark.parametrize("rows,heads,kvh", [(127, 80, 80), (128, 80, 80), (129, 80, 80), (127, 80, 40), (128, 80, 40),
                                            (129, 80, 40), (255, 40, 40), (256, 40, 40), (257, 40, 40), (255, 80, 40)])
def test_rows_around_the_tiles(be, dtype, hd, rows, heads, kvh):
    c = Cache([rows + 250], kvh, hd, seed=rows)
    check(be, c, [0, rows], [rows + 250], heads, dtype, "prompt")


@pytest.mark.parametrize("dtype,hd", [("f16", 64), ("bf16", 64), ("f16", 128), ("bf16", 128)])
def test_equal_prompts(be, dtype, hd):
    """The whole batch by one launch; one sequence has more context than rows, one padding rows, one is a free slot."""
    ctx = [400, 1000, 401, 390, 0]
    c = Cache(ctx, 8, hd, seed=2)
    check(be, c, [0, 400, 800, 1200, 1600, 2000], ctx, 32, dtype, "prompt", "odd")


@pytest.mark.parametrize("dtype,hd", [("f16", 64), ("bf16", 64), ("f16", 128), ("bf16", 128)])
@pytest.mark.parametrize("heads,kvh", [(40, 8), (9, 9), (21, 3)])
def test_prompts_among_single_tokens(be, dtype, hd, heads, kvh):
    n = [1, 700, 0, 1, 64, 1, 1100, 13, 65, 1]
    ctx = [1, 900, 7, 0, 64, 1300, 1100, 500, 600, 17]
    starts = [0]
    for i in n:
        starts.append(starts[-1] + i)
    c = Cache(ctx, kvh, hd, seed=4)
    check(be, c, starts, ctx, heads, dtype, "both")


@pytest.mark.parametrize("dtype,hd", [("f16", 64), ("bf16", 128)])
def test_scores_far_apart_and_scales_far_apart(be, dtype, hd):
    """Large queries put all the weight on few tokens; pages whose scales differ by 10^6; scales of zero."""
    ctx = [1000, 1100]
    starts = [0, 900, 1800]
    c = Cache(ctx, 8, hd, seed=11)
    check(be, c, starts, ctx, 32, dtype, "prompt", gain=30.0, norm=False)
    c.scales[c.tab[0, 3].item(), :, 1] *= 1e6
    c.scales[c.tab[0, 5].item(), :, 1] *= 1e-6
    c.scales[c.tab[0, 9].item(), :, 0] = 0.0
    c.scales[c.tab[1, 2].item(), :, :] = 0.0
    check(be, c, starts, ctx, 32, dtype, "prompt", norm=False)
    check(be, c, starts, ctx, 32, dtype, "prompt", scale=0.01, norm=False)


def tensors(rows, heads, hd, dtype):
    q = torch.randn(rows, heads, hd, generator=torch.Generator(device="cuda").manual_seed(3), device="cuda")
    q = q.to(TYPES[dtype][0])
    return q, torch.empty_like(q)


@pytest.mark.parametrize("dtype,hd", [("f16", 128), ("bf16", 64)])
def test_what_no_row_sees_does_not_count(be, dtype, hd):
    """NaN and infinite scales in pages past the context, and in a page that only later rows see."""
    c = Cache([1000], 8, hd, seed=2)
    q, ref = tensors(800, 32, hd, dtype)
    out = torch.empty_like(ref)
    run(be, c, [0, 800], [900], q, ref, 32, "prompt", dtype)
    be.synchronize()
    assert bool(torch.isfinite(ref).all())
    c.scales[c.tab[0, 57:62].long()] = float("nan")   # tokens 912 .. 991: past the context
    c.scales[c.tab[0, 62].item()] = float("inf")
    c.scales[c.tab[0, 56].item()] = float("inf")      # tokens 896 .. 899: seen by the last four rows only
    run(be, c, [0, 800], [900], q, out, 32, "prompt", dtype)
    be.synchronize()
    assert torch.equal(out[:796], ref[:796])
    assert not bool(torch.isfinite(out[796:]).all(-1).any())
    c.scales[c.tab[0, 56].item()] = float("nan")
    run(be, c, [0, 800], [900], q, out, 32, "prompt", dtype)
    be.synchronize()
    assert torch.equal(out[:796], ref[:796]) and bool(torch.isnan(out[796:]).all())


@pytest.mark.parametrize("dtype,hd", [("f16", 64), ("bf16", 128)])
def test_queries_that_are_not_finite_keep_to_their_rows(be, dtype, hd):
    c = Cache([1000], 8, hd, seed=2)
    q, ref = tensors(1000, 32, hd, dtype)
    out = torch.empty_like(ref)
    run(be, c, [0, 1000], [1000], q, ref, 32, "prompt", dtype)
    q[300, 7, 5], q[999, 31, hd - 1], q[500, 0, 0] = float("nan"), float("inf"), float("-inf")
    run(be, c, [0, 1000], [1000], q, out, 32, "prompt", dtype)
    be.synchronize()
    hit = torch.zeros(1000, 32, dtype=torch.bool, device="cuda")
    hit[300, 7] = hit[999, 31] = hit[500, 0] = True
    assert torch.equal(out[~hit], ref[~hit]) and bool(torch.isnan(out[hit]).all())


@pytest.mark.parametrize("dtype,hd", [("f16", 128), ("bf16", 64)])
@pytest.mark.parametrize("page", [-1, "past", 2 ** 31 - 1])
def test_a_page_out_of_range_is_left_out_and_reported(be, dtype, hd, page):
    ctx = [800, 900]
    c = Cache(ctx, 8, hd, seed=6)
    q, out = tensors(1600, 32, hd, dtype)
    c.tab[1, 20] = c.blocks if page == "past" else page
    run(be, c, [0, 800, 1600], ctx, q, out, 32, "prompt", dtype)
    with pytest.raises(L.PoxError, match="block-table entry"):
        be.synchronize()
    ref, mag, vmax, e = formula(c, [0, 800, 1600], ctx, q, 1 / math.sqrt(hd), without=[(1, 20)])
    u = TYPES[dtype][2]
    tol = (2.0 ** -11 + 2 * e + 2.0 ** -16) * mag + 900 * 2.0 ** -25 * vmax + 1.01 * u * ref.abs() + 2.0 ** -24
    assert bool(((out.double() - ref).abs() <= tol).all())


@pytest.mark.parametrize("dtype,hd", [("f16", 64), ("bf16", 128)])
def test_bounds_that_a_prompt_breaks_are_reported(be, dtype, hd):
    ctx = [800, 900]
    c = Cache(ctx, 8, hd, seed=6)
    q, good = tensors(1600, 32, hd, dtype)
    out = torch.empty_like(good)
    run(be, c, [0, 800, 1600], ctx, q, good, 32, "prompt", dtype)
    be.synchronize()
    b = c.batch([0, 800, 1600], ctx)
    b.max_ctx = 899
    out.fill_(7.0)
    be.kv8_attention(c.c, b, rows_of(q), rows_of(out), 32, 0.0, STREAM)
    with pytest.raises(L.PoxError, match="bounds"):
        be.synchronize()
    assert torch.equal(out[:800], good[:800]) and bool((out[800:] == 7.0).all())


def test_f32_prompts_take_the_step_kernel(be):
    assert route([0, 1000], 1000, 1000, 32, 8, 128, "f32") == "step"
    assert route([0, 1000], 1000, 1000, 32, 8, 32, "f16") == "step"
