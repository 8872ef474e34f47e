"""The 8-bit paged KV cache where its calls can go wrong: magnitudes at the ends of f32, streams that share a handle,
row starts that do not describe the rows, positions outside the rotation table, launches past the grid's limit, first
calls before a capture.

Stored bytes and scales follow the rule element by element in f32, so they are compared for equality with its numpy
restatement (test_kv8_gpu.np_append)."""
import ctypes
import threading

import numpy as np
import pytest
from test_kv8_gpu import STREAM, Cache, np_append, rope_table, rows_of

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


def check_append(be, c, starts, ctx, k, v):
    pages, scales = c.pages.cpu().numpy(), c.scales.cpu().numpy()
    with np.errstate(all="ignore"):
        np_append(pages, scales, c, c.tab_np, starts, ctx, k.float().cpu().numpy(), v.float().cpu().numpy(), None, 0,
                  False)
    be.kv8_append(c.c, c.batch(starts, ctx), rows_of(k), rows_of(v), None, STREAM)
    be.synchronize()
    assert np.array_equal(c.scales.cpu().numpy(), scales, equal_nan=True)
    used = [b for s, x in enumerate(ctx) for b in c.tab_np[s, :(x + 15) // 16]]
    assert np.array_equal(c.pages.cpu().numpy()[used], pages[used])


# largest magnitudes of a page, in units of 2^-149: around the steps of the rounded scale m / 127
SMALL = [1, 63, 64, 100, 127, 128, 150, 189, 190, 191, 254, 317, 318, 1000, 16129, 16192, 2 ** 22, 2 ** 23 - 1, 2 ** 23]


@pytest.mark.parametrize("hd", [32, 64, 128])
@pytest.mark.parametrize("most", SMALL)
def test_append_of_subnormal_magnitudes(be, hd, most):
    rng = np.random.default_rng(most)
    n = 21
    units = rng.integers(-most, most + 1, size=(2, n, 2, hd))
    units[:, ::5, :, 3], units[:, 1::5, :, hd - 1] = most, -most
    sign = (units < 0).astype(np.uint32) << np.uint32(31)
    x = (np.abs(units).astype(np.uint32) | sign).view(np.float32)
    k, v = (torch.from_numpy(a.copy()).cuda() for a in x)
    c = Cache([n], 2, hd, fill=False)
    check_append(be, c, [0, 17], [17], k[:17].contiguous(), v[:17].contiguous())
    check_append(be, c, [0, 4], [21], k[17:].contiguous(), v[17:].contiguous())  # onto older slots of such a page


@pytest.mark.parametrize("size", [2.0 ** -126, 2.0 ** -100, 2.0 ** -91, 2.0 ** -90, 2.0 ** -64, 2.0 ** -57, 2.0 ** 57,
                                  2.0 ** 71, 2.0 ** 119, 2.0 ** 120, 2.0 ** 125])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_append_where_a_scale_s_reciprocal_leaves_the_range(be, dtype, size):
    dt = torch.float32 if dtype == "f32" else torch.bfloat16
    g = torch.Generator(device="cuda").manual_seed(3)
    k, v = (torch.randn(40, 3, 64, generator=g, device="cuda").clamp(-5, 5).mul(size).to(dt) for _ in range(2))
    v[7, 1, 2], v[9, 0, 0], v[11, 2, 63] = float("inf"), float("-inf"), float("nan")
    c = Cache([40], 3, 64, fill=False)
    check_append(be, c, [0, 21], [21], k[:21], v[:21])
    check_append(be, c, [0, 1], [22], k[21:22] * 2, v[21:22] * 0.5)  # the older slots of one side follow
    check_append(be, c, [0, 18], [40], k[22:], v[22:])


def test_append_of_small_rows_onto_large_pages_and_back(be):
    """A page whose scale is huge takes rows of nothing, and the other way round."""
    c = Cache([16], 1, 64, fill=False)
    one = torch.ones(1, 1, 64, device="cuda")
    for i, power in enumerate([-149, -140, -120, -60, 0, 60, 126, -149]):
        x = one * 2.0 ** power * 1.25
        check_append(be, c, [0, 1], [i + 1], x, -x)


class Steps:
    """Single tokens over long contexts, which the GPU splits and joins through the stream's partials."""

    def __init__(self, seed, ctx):
        g = torch.Generator(device="cuda").manual_seed(seed)
        self.c = Cache(ctx, 2, 64, seed=seed)
        self.b = self.c.batch(list(range(len(ctx) + 1)), ctx)
        self.q = torch.randn(len(ctx), 8, 64, generator=g, device="cuda")

    def attend(self, be, out, stream):
        be.kv8_attention(self.c.c, self.b, rows_of(self.q), rows_of(out), 8, 0.0, stream)


def test_threads_on_the_per_thread_stream_have_partials_of_their_own(be):
    per_thread = 2  # cudaStreamPerThread: one handle, a stream of each thread
    work = [Steps(1, [30001, 9000]), Steps(2, [12345, 4567, 20000])]
    want = [torch.empty_like(w.q) for w in work]
    outs = [[torch.empty_like(w.q) for _ in range(200)] for w in work]
    for w, o in zip(work, want):
        w.attend(be, o, STREAM)
    be.synchronize()
    errors, gate = [], threading.Barrier(2)

    def run(i):
        try:
            gate.wait()
            for o in outs[i]:
                work[i].attend(be, o, per_thread)
            be.synchronize()  # (the stream ends with the thread)
        except Exception as e:  # noqa: BLE001
            errors.append(e)

    threads = [threading.Thread(target=run, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    be.synchronize()
    assert not errors
    for o, w in zip(outs, want):
        assert all(torch.equal(x, w) for x in o)


def test_streams_that_come_and_go(be):
    """Streams that are destroyed after their work (the driver gives handles out again): right results, and partials
    that are taken over instead of piling up."""
    cuda = ctypes.CDLL("libcuda.so.1")
    w = Steps(3, [50000, 31000])
    want = torch.empty_like(w.q)
    w.attend(be, want, STREAM)
    be.synchronize()
    handles, free = set(), None
    for i in range(12):
        outs = [torch.empty_like(w.q) for _ in range(8)]
        torch.cuda.synchronize()
        streams = [ctypes.c_void_p() for _ in outs]
        for o, s in zip(outs, streams):
            assert cuda.cuStreamCreate(ctypes.byref(s), 1) == 0
            w.attend(be, o, s.value)
            w.attend(be, o, s.value)
        be.synchronize()
        for s in streams:
            assert cuda.cuStreamDestroy_v2(s) == 0
            handles.add(s.value)
        assert all(torch.equal(o, want) for o in outs)
        if i == 5:
            free = torch.cuda.mem_get_info()[0]
    if len(handles) < 48:  # handles did come back
        assert torch.cuda.mem_get_info()[0] > free - 64 * 2 ** 20


# row starts, rows, the bound of a sequence's rows, sequences left out
STARTS = [
    ([0, 2, 2], 2, 1, [0, 1]),       # as many rows as sequences, at most one each, but not one each
    ([1, 1, 2], 2, 1, [0]),
    ([0, 1, 2, 2], 3, 1, [2]),       # the third row belongs to no sequence
    ([3, 6, 9], 9, 3, [0]),          # the first rows belong to none
    ([20, 60, 90], 90, 60, [0]),
    ([0, 3, 7], 9, 4, [1]),          # nor the last
]


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("starts,rows,most,out_of", STARTS)
def test_row_starts_that_do_not_fit_are_reported_and_left_out(be, dtype, starts, rows, most, out_of):
    dt = torch.float32 if dtype == "f32" else torch.bfloat16
    seqs = len(starts) - 1
    ctx = [50 + 40 * s + most for s in range(seqs)]
    c = Cache(ctx, 2, 64, seed=rows)
    b = c.batch(starts, ctx)
    b.row_starts, b.rows, b.max_rows = c.keep[0].data_ptr(), rows, most
    g = torch.Generator(device="cuda").manual_seed(1)
    q, k, v = (torch.randn(rows, h, 64, generator=g, device="cuda").to(dt) for h in (4, 2, 2))
    out, ko, vo = (torch.full_like(t, 7.0) for t in (q, k, v))
    kept = [s for s in range(seqs) if s not in out_of]
    own = torch.zeros(rows, dtype=torch.bool)
    for s in kept:
        own[starts[s]:starts[s + 1]] = True
    before = c.pages.clone(), c.scales.clone()
    for call in (lambda: be.kv8_attention(c.c, b, rows_of(q), rows_of(out), 4, 0.0, STREAM),
                 lambda: be.kv8_read(c.c, b, rows_of(ko), rows_of(vo), STREAM),
                 lambda: be.kv8_append(c.c, b, rows_of(k), rows_of(v), None, STREAM)):
        call()
        with pytest.raises(L.PoxError, match="bounds"):
            be.synchronize()
    for t in (out, ko, vo):
        assert bool((t[~own] == 7.0).all()) and not bool((t[own] == 7.0).all(-1).any())
    for s in range(seqs):
        blocks = torch.from_numpy(c.tab_np[s, :(ctx[s] + 15) // 16].astype(np.int64)).cuda()
        same = torch.equal(c.pages[blocks], before[0][blocks]) and torch.equal(c.scales[blocks], before[1][blocks])
        assert same == (s in out_of)


@pytest.mark.parametrize("rows,starts", [(3000, [100, 3000]), (3000, [0, 2900])])
def test_row_starts_of_a_prompt_that_do_not_fit(be, rows, starts):
    c = Cache([3000], 8, 128, seed=1)
    b = c.batch(starts, [3000])
    b.row_starts, b.rows, b.max_rows = c.keep[0].data_ptr(), rows, rows
    q = torch.randn(rows, 32, 128, device="cuda").half()
    out = torch.full_like(q, 7.0)
    be.kv8_attention(c.c, b, rows_of(q), rows_of(out), 32, 0.0, STREAM)
    with pytest.raises(L.PoxError, match="bounds"):
        be.synchronize()
    assert bool((out == 7.0).all())


@pytest.mark.parametrize("dtype,rot,half,pad", [("bf16", 64, True, 0), ("f32", 64, False, 0), ("f16", 6, True, 0),
                                                ("f32", 64, True, 1)])
def test_append_outside_the_rotation_table_leaves_the_page(be, dtype, rot, half, pad):
    """Pages of slots 0 and later, and one that holds older tokens; `pad` takes the rows off the vector loads."""
    dt = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}[dtype]
    ctx, starts, positions = [50, 20, 40], [0, 40, 43, 47], 36
    c = Cache(ctx, 2, 64, seed=5)
    table = rope_table(positions, rot)
    rope = L.Rope(table.data_ptr(), positions, rot, L.POX_ROPE_HALF if half else L.POX_ROPE_INTERLEAVED)
    k, v = (torch.randn(47, 2, 64 + pad, device="cuda").mul(9).to(dt)[..., :64] for _ in range(2))
    before, scales = c.pages.clone(), c.scales.clone()
    be.kv8_append(c.c, c.batch(starts, ctx), rows_of(k), rows_of(v), rope, STREAM)
    with pytest.raises(L.PoxError, match="rotation table"):
        be.synchronize()
    # sequence 0 takes tokens 10 .. 49, 1 takes 17 .. 19, 2 takes 36 .. 39: pages whose last new row is past 35 stay
    changed = {(0, 0), (0, 1), (1, 1)}
    for s, x in enumerate(ctx):
        for page in range((x + 15) // 16):
            b = c.tab_np[s, page]
            for side in range(2):
                same = torch.equal(c.scales[b, :, side], scales[b, :, side])
                half_page = slice(16 * 64 * side, 16 * 64 * (side + 1))
                same = same and torch.equal(c.pages[b, :, half_page], before[b, :, half_page])
                assert same == ((s, page) not in changed), (s, page, side)


@pytest.mark.parametrize("dtype,heads,hd", [("bf16", 64, 128), ("f32", 40, 64), ("f16", 9, 96)])
def test_norms_at_positions_outside_the_table_leave_their_rows(be, dtype, heads, hd):
    """Rows whose loads are on their way when the position is looked at; the rows around them are as without them."""
    dt = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}[dtype]
    g = torch.Generator(device="cuda").manual_seed(2)
    x = torch.randn(500, heads, hd, generator=g, device="cuda").to(dt)
    good, y = torch.zeros_like(x), torch.full_like(x, 7.0)
    w = torch.ones(hd, device="cuda").half()
    table = rope_table(600, hd)
    pos = torch.arange(500, device="cuda", dtype=torch.int32)

    def call(out, positions):
        rope = L.Rope(table.data_ptr(), positions, hd, L.POX_ROPE_HALF)
        be.qk_norm_rope(L.QkNormRope(rows_of(x), L.Rows(), rows_of(out), L.Rows(), 500, heads, 0, hd, w.data_ptr(), 0,
                                     1e-5, rope, pos.data_ptr()), STREAM)

    call(good, 600)
    be.synchronize()
    call(y, 333)
    with pytest.raises(L.PoxError, match="rotation table"):
        be.synchronize()
    assert torch.equal(y[:333], good[:333]) and bool((y[333:] == 7.0).all())


@pytest.mark.parametrize("rows,heads,hd", [(2 ** 26, 4096, 2), (2 ** 26, 513, 2), (2 ** 26, 2047, 512)])
def test_norms_of_more_heads_than_a_launch_holds_are_refused(be, rows, heads, hd):
    """(refused on the host: the sizes are the views' own, no memory of that size stands behind them)"""
    x = torch.zeros(16, device="cuda", dtype=torch.half)
    view = L.Rows(x.data_ptr(), L.POX_F16, heads * hd, hd)
    args = L.QkNormRope(view, view, view, view, rows, heads, heads, hd, 0, 0, 1e-5, L.Rope(), 0)
    with pytest.raises(L.PoxError):
        be.qk_norm_rope(args, STREAM)
    be.synchronize()


def test_any_first_call_readies_a_stream_for_capture(be):
    """A prompt without the step kernel, then a captured decode step; and a captured prompt as a first call."""
    c = Cache([1000], 8, 64, seed=1)
    q = torch.randn(1000, 32, 64, device="cuda").bfloat16()
    out, eager, last, want = (torch.empty_like(q[:n]) for n in (1000, 1000, 1, 1))
    prompt, step = c.batch([0, 1000], [1000]), c.batch([0, 1], [1000])
    be.kv8_attention(c.c, prompt, rows_of(q), rows_of(eager), 32, 0.0, STREAM)
    be.kv8_attention(c.c, step, rows_of(q[999:]), rows_of(want), 32, 0.0, STREAM)
    torch.cuda.synchronize()
    st, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    be.kv8_attention(c.c, prompt, rows_of(q), rows_of(out), 32, 0.0, st.cuda_stream)
    torch.cuda.synchronize()
    assert torch.equal(out, eager)
    with torch.cuda.graph(graph, stream=st):
        be.kv8_attention(c.c, step, rows_of(q[999:]), rows_of(last), 32, 0.0, st.cuda_stream)
    graph.replay()
    be.synchronize()
    assert torch.equal(last, want)
    st, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    out.zero_()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=st):
        be.kv8_attention(c.c, prompt, rows_of(q), rows_of(out), 32, 0.0, st.cuda_stream)
    graph.replay()
    be.synchronize()
    assert torch.equal(out, eager)
