"""Cases of the 8-bit KV-cache operators: what is measured, their plain forms and their definition in 64 bits.

Three operators of a serving step, in the order in which a layer calls them after its q/k/v projection:

  qk      per-head RMSNorm of q and k with the position rotation in the same pass (CudaBackend.qk_norm_rope)
  append  new k and v rows into pages of 16 tokens held in 8 bits, one f32 scale for each page, kv head and side, k
          rotated on the way (CudaBackend.kv8_append); the pass then reads back the live rows of every page that it
          touched (CudaBackend.kv8_read), so that the cache's new state comes out as the values that it stands for
  attend  attention of new rows over those pages: single tokens, prompt chunks and mixtures (CudaBackend.kv8_attention)

Row i of the n rows of a sequence with ctx tokens in the cache (its new ones included) stands at position ctx - n + i
and sees the positions up to its own; a row of a negative position is padding and sees nothing (its output is 0).

A page of one kv head is 32 * head_dim bytes: K of token t, dim d at t * hd + (d ^ 64 if hd == 128 and t is odd else d),
then V of token t, dim d at 16 * hd + 16 * d + t.
"""
import math

import torch

own = False

PAGE = 16
DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
ESIZE = {"f32": 4, "f16": 2, "bf16": 2}


# ---- the cases ----------------------------------------------------------------------------------------------------
def listed():
    return [
        # one decode step of one sequence, this framework's own f32 rows of an 8B-class layer: latency is all there is
        dict(name="qk step b1 f32", op="qk", rows=1, heads=32, kv_heads=8, hd=128, rot=128, half=False, norm=True,
             dtype="f32", fused=True),
        # a small odd batch of an MHA model with a partial rotation, q and k in buffers of their own, head-major
        dict(name="qk 517 rows f16", op="qk", rows=517, heads=16, kv_heads=16, hd=64, rot=32, half=True, norm=True,
             dtype="f16", fused=False),
        # a pass of prompts of a 70B-class layer, q and k inside the projection's output rows
        dict(name="qk 16384 rows bf16", op="qk", rows=16384, heads=64, kv_heads=8, hd=128, rot=128, half=True,
             norm=True, dtype="bf16", fused=True),
        # a decode step of 64 sequences: one row each, nearly every one into a page that holds older tokens
        dict(name="append step b64 bf16", op="append", seqs=64, rows_lo=1, rows_hi=1, ctx_lo=3900, ctx_hi=4300, pad=0,
             kv_heads=8, hd=128, rot=128, half=True, dtype="bf16"),
        # prompt chunks of several sequences at once, ragged, most of them starting inside a page
        dict(name="append ragged f16", op="append", seqs=23, rows_lo=1, rows_hi=700, ctx_lo=700, ctx_hi=2100, pad=0,
             kv_heads=12, hd=64, rot=32, half=True, dtype="f16"),
        # one long prompt from an empty cache, in this framework's f32 rows and interleaved rotation
        dict(name="append prompt f32", op="append", seqs=1, rows_lo=16381, rows_hi=16381, ctx_lo=16381, ctx_hi=16381,
             pad=0, kv_heads=8, hd=128, rot=128, half=False, dtype="f32"),
        # one decode step of one sequence at the context of this framework's decode benchmark: latency
        dict(name="attend step b1 f32", op="attend", seqs=1, rows_lo=1, rows_hi=1, ctx_lo=640, ctx_hi=640, pad=0,
             heads=32, kv_heads=8, hd=128, dtype="f32"),
        # a decode step of a batch of an MHA model, short and long contexts, some slots of the batch empty
        dict(name="attend step b37 f16", op="attend", seqs=37, rows_lo=1, rows_hi=1, ctx_lo=1, ctx_hi=2011, pad=4,
             heads=12, kv_heads=12, hd=64, dtype="f16"),
        # the batch and context of this framework's 70B decode benchmark
        dict(name="attend step b64 bf16", op="attend", seqs=64, rows_lo=1, rows_hi=1, ctx_lo=3800, ctx_hi=4400, pad=0,
             heads=64, kv_heads=8, hd=128, dtype="bf16"),
        # few sequences of a long context: the context has to be split to fill the GPU
        dict(name="attend long b3 f16", op="attend", seqs=3, rows_lo=1, rows_hi=1, ctx_lo=40000, ctx_hi=131000, pad=0,
             heads=32, kv_heads=8, hd=128, dtype="f16"),
        # chunks of prompts next to decoding sequences in one pass, seven query heads to a kv head, f32 rows
        dict(name="attend mixed f32", op="attend", seqs=20, rows_lo=1, rows_hi=257, ctx_lo=300, ctx_hi=5000, pad=1,
             heads=14, kv_heads=2, hd=64, dtype="f32"),
        # one long prompt: the products bound it
        dict(name="attend prompt bf16", op="attend", seqs=1, rows_lo=8192, rows_hi=8192, ctx_lo=8192, ctx_hi=8192,
             pad=0, heads=32, kv_heads=8, hd=128, dtype="bf16"),
    ]


def _log(rng, lo, hi):
    n = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    return n + (n == 3072)


def draw(rng):
    op = rng.choice(["qk", "append", "attend", "attend"])
    hd = rng.choice([64, 128, 128])
    dtype = rng.choice(["f32", "f16", "bf16"])
    kv_heads, group = rng.choice([(8, 4), (8, 8), (2, 7), (12, 1), (4, 5), (1, 6), (16, 2)])
    if op == "qk":
        most = (16384 * 72 * 128 * 2) // ((kv_heads * (group + 1)) * hd * ESIZE[dtype])
        return dict(op=op, rows=_log(rng, 1, min(most, 16384)), heads=kv_heads * group, kv_heads=kv_heads, hd=hd,
                    rot=rng.choice([hd, hd, hd // 2]), half=rng.random() < 0.5, norm=rng.random() < 0.7, dtype=dtype,
                    fused=rng.random() < 0.6)
    if op == "append":
        rot, half = rng.choice([hd, hd, hd // 2, 0]), rng.random() < 0.5
        if rng.random() < 0.4:  # a decode step
            seqs, lo, hi, ctx_lo = _log(rng, 1, 128), 1, 1, rng.randint(1, 100)
            ctx_hi = _log(rng, 200, 5000)
        else:
            total = _log(rng, 40, 16000)
            seqs = _log(rng, 1, min(32, total))
            hi = max(1, total // seqs)
            lo, ctx_lo = rng.choice([1, hi]), hi
            ctx_hi = ctx_lo + rng.choice([0, _log(rng, 1, 2000)])
        if kv_heads > 8:
            kv_heads = 8
        return dict(op=op, seqs=seqs, rows_lo=lo, rows_hi=hi, ctx_lo=ctx_lo, ctx_hi=ctx_hi, pad=rng.choice([0, 0, 1]),
                    kv_heads=kv_heads, hd=hd, rot=rot, half=half, dtype=dtype)
    heads = kv_heads * group
    kind = rng.choice(["step", "step", "few", "chunk"])
    if kind == "few":  # few sequences of a long context; a cache of at most 0.5 GB
        seqs, lo, hi = rng.randint(1, 4), 1, rng.choice([1, 1, 2, 4])
        ctx_hi = min(_log(rng, 4000, 131000), (1 << 28) // (seqs * kv_heads * hd))
        ctx_lo = max(4, ctx_hi // rng.choice([1, 2, 8]))
    elif kind == "step":
        seqs, lo, hi = _log(rng, 1, 128), 1, rng.choice([1, 1, 1, 3])
        ctx_hi = max(8, min(_log(rng, 16, 8000), (1 << 28) // (seqs * kv_heads * hd)))
        ctx_lo = rng.randint(4, ctx_hi)
    else:  # prompt chunks: rows times context bounded by the largest listed case
        hi = _log(rng, 17, 6000)
        seqs = _log(rng, 1, max(1, min(32, 6000 // hi)))
        lo = rng.choice([1, hi])
        ctx_hi = max(hi, min(hi + _log(rng, 1, 6000), (8192 * 8192 * 32) // (2 * hi * seqs * heads)))
        ctx_lo = max(hi, ctx_hi // 2)
    return dict(op=op, seqs=seqs, rows_lo=lo, rows_hi=hi, ctx_lo=ctx_lo, ctx_hi=ctx_hi, pad=rng.choice([0, 0, 1]),
                heads=heads, kv_heads=kv_heads, hd=hd, dtype=dtype)


def _lens(c):
    """(rows, context) of each sequence: spread over the case's ranges by the golden ratio, so that they are the case's
    own and not the seed's; the last `pad` sequences are empty slots (one row, no context)."""
    n, s = c["seqs"], []
    for i in range(n):
        u, w = (0.5 + i * 0.6180339887498949) % 1.0, (0.25 + i * 0.7548776662466927) % 1.0
        # two thirds of a ragged batch are single tokens, the rest spread up to rows_hi
        rows = c["rows_hi"] if c["rows_lo"] == c["rows_hi"] else 1 if i % 3 else c["rows_lo"] + int(
            (c["rows_hi"] - c["rows_lo"]) * (1.0 if i == 0 else u))
        ctx = c["ctx_lo"] + int((c["ctx_hi"] - c["ctx_lo"]) * (1.0 if i == 0 else w))
        s.append((rows, max(ctx, rows)))
    return s + [(1, 0)] * c["pad"]


def work(c):
    es, hd = ESIZE[c["dtype"]], c["hd"]
    if c["op"] == "qk":
        n = c["rows"] * (c["heads"] + c["kv_heads"]) * hd
        return {"bytes": 2 * n * es + c["rows"] * (4 + 4 * c["rot"]) + 4 * hd, "flops": n * (4 * c["norm"] + 3)}
    lens, kvh = _lens(c), c["kv_heads"]
    if c["op"] == "append":  # rows in, their bytes written, the touched pages' older bytes read, the live rows out
        new = sum(r for r, x in lens if x)
        live = sum(x - (x - r) // PAGE * PAGE for r, x in lens if x)
        return {"bytes": 2 * kvh * hd * (new * es + new + (live - new) + live * es) + 4 * c["rot"] * new,
                "flops": 2 * kvh * hd * new * 6}
    rows, heads = sum(r for r, _ in lens), c["heads"]
    seen = sum(r * x - r * (r - 1) // 2 for r, x in lens if x)
    pages = sum(-(-x // PAGE) for _, x in lens)
    return {"bytes": 2 * rows * heads * hd * es + sum(x for _, x in lens) * kvh * hd * 2 + pages * kvh * 8 + 4 * pages,
            "flops": 4 * hd * heads * seen}


# ---- what a program has in hand -----------------------------------------------------------------------------------
def _rope_table(positions, rot):
    """(cos, sin) of each position and pair, f32 [positions][rot / 2][2], base 500000 (the framework's default)."""
    inv = 500000.0 ** (-torch.arange(0, rot, 2, dtype=torch.float64, device="cuda") / rot)
    a = torch.arange(positions, dtype=torch.float64, device="cuda")[:, None] * inv
    return torch.stack([a.cos(), a.sin()], -1).float().contiguous()


def _rows(g, rows, heads, hd, dtype):
    """Projected rows: normal, each head with a scale of its own and a few dims several times larger."""
    x = torch.randn(rows, heads, hd, generator=g, device="cuda")
    x *= 0.5 + torch.rand(1, heads, 1, generator=g, device="cuda") * 2
    x[..., 5::31] *= 4
    return x.to(dtype)


def prepare(c, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    dt, hd, s = DTYPES[c["dtype"]], c["hd"], dict(c)
    if c["op"] == "qk":
        rows, h, kvh = c["rows"], c["heads"], c["kv_heads"]
        if c["fused"]:  # q and k are slices of the projection's output rows (q | k | v); the results go to such a row too
            x = torch.empty(rows, h + 2 * kvh, hd, dtype=dt, device="cuda")
            x.copy_(_rows(g, rows, h + 2 * kvh, hd, dt))
            y = torch.empty(rows, h + kvh, hd, dtype=dt, device="cuda")
            s.update(q=x[:, :h], k=x[:, h:h + kvh], q_out=y[:, :h], k_out=y[:, h:])
        else:  # buffers of their own, one head after the other
            s.update(q=_rows(g, rows, h, hd, dt).transpose(0, 1).contiguous().transpose(0, 1),
                     k=_rows(g, rows, kvh, hd, dt).transpose(0, 1).contiguous().transpose(0, 1))
            s.update(q_out=torch.empty_like(s["q"]), k_out=torch.empty_like(s["k"]))
        s["q_norm"] = (1 + 0.2 * torch.randn(hd, generator=g, device="cuda")).half() if c["norm"] else None
        s["k_norm"] = (1 + 0.2 * torch.randn(hd, generator=g, device="cuda")).half() if c["norm"] else None
        table = max(rows, 4096)
        s["table"] = _rope_table(table, c["rot"])
        s["positions"] = torch.randint(0, table, (rows,), generator=g, device="cuda", dtype=torch.int32)
    else:
        lens, kvh = _lens(c), c["kv_heads"]
        starts = [0]
        for r, _ in lens:
            starts.append(starts[-1] + r)
        rows, most = starts[-1], max(x for _, x in lens)
        width = -(-most // PAGE) + 1
        need = [-(-x // PAGE) for _, x in lens]
        blocks = sum(need) + 3
        perm = torch.randperm(blocks, generator=g, device="cuda", dtype=torch.int32)
        tab = torch.full((len(lens), width), -1, dtype=torch.int32, device="cuda")
        at = 0
        for i, n in enumerate(need):
            tab[i, :n] = perm[at:at + n]
            at += n
        # the cache: quantised normal values (3.5 sigma at the end of the range), scales that differ from page to page
        pages = torch.empty(blocks, kvh, 32 * hd, dtype=torch.int8, device="cuda")
        step = max(1, (1 << 26) // (kvh * 32 * hd))
        for b in range(0, blocks, step):
            part = pages[b:b + step]
            part.copy_(torch.randn(part.shape, generator=g, device="cuda").mul_(36).round_().clamp_(-127, 127))
        scales = torch.rand(blocks, kvh, 2, generator=g, device="cuda").mul_(0.6).exp_().mul_(0.02)
        i32 = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
        s.update(pages=pages, scales=scales, tables=tab, row_starts=i32(starts), ctx=i32([x for _, x in lens]),
                 rows=rows, max_rows=max(r for r, _ in lens), max_ctx=most, n=len(lens))
        if c["op"] == "append":
            s.update(k=_rows(g, rows, kvh, hd, dt), v=_rows(g, rows, kvh, hd, dt))
            s["table"] = _rope_table(most, c["rot"]) if c["rot"] else None
            live = [x - (x - r) // PAGE * PAGE if x else 0 for r, x in lens]
            ends = [0]
            for n in live:
                ends.append(ends[-1] + n)
            s.update(read_starts=i32(ends), read_rows=ends[-1], read_max=max(live))
            s.update(k_out=torch.empty(ends[-1], kvh, hd, dtype=dt, device="cuda"),
                     v_out=torch.empty(ends[-1], kvh, hd, dtype=dt, device="cuda"))
        else:
            s.update(q=_rows(g, rows, c["heads"], hd, dt), out=torch.empty(rows, c["heads"], hd, dtype=dt, device="cuda"))
    if own:  # the framework's handles of those tensors: addresses, sizes and strides, as a program keeps them
        s["call"] = _call(s)
    return s


# ---- the framework's operators ------------------------------------------------------------------------------------
_backend = None


def _call(s):
    global _backend
    from paraoxidizer_b200 import _lib as L
    from paraoxidizer_b200.backend import CudaBackend

    if _backend is None:
        _backend = CudaBackend.create(0)
    code = {torch.float32: L.POX_F32, torch.float16: L.POX_F16, torch.bfloat16: L.POX_BF16}
    view = lambda t: L.Rows(t.data_ptr(), code[t.dtype], t.stride(0), t.stride(1))  # noqa: E731
    style = L.POX_ROPE_HALF if s.get("half") else L.POX_ROPE_INTERLEAVED
    rope = None
    if s.get("table") is not None:
        rope = L.Rope(s["table"].data_ptr(), s["table"].shape[0], s["rot"], style)
    if s["op"] == "qk":
        ptr = lambda t: 0 if t is None else t.data_ptr()  # noqa: E731
        return (L.QkNormRope(view(s["q"]), view(s["k"]), view(s["q_out"]), view(s["k_out"]), s["rows"], s["heads"],
                             s["kv_heads"], s["hd"], ptr(s["q_norm"]), ptr(s["k_norm"]), 1e-5, rope,
                             s["positions"].data_ptr()),)
    cache = L.Kv8Cache(s["pages"].data_ptr(), s["scales"].data_ptr(), s["pages"].shape[0], s["kv_heads"], s["hd"])
    batch = lambda starts, rows, most: L.Kv8Batch(  # noqa: E731
        starts.data_ptr(), s["ctx"].data_ptr(), s["tables"].data_ptr(), s["n"], rows, most, s["max_ctx"],
        s["tables"].shape[1])
    if s["op"] == "append":
        return (cache, batch(s["row_starts"], s["rows"], s["max_rows"]), view(s["k"]), view(s["v"]), rope,
                batch(s["read_starts"], s["read_rows"], s["read_max"]), view(s["k_out"]), view(s["v_out"]))
    return cache, batch(s["row_starts"], s["rows"], s["max_rows"]), view(s["q"]), view(s["out"]), s["heads"]


def run(s):
    if not own:
        return {"qk": _plain_qk, "append": _plain_append, "attend": _plain_attend}[s["op"]](s)
    be, a = _backend, s["call"]
    stream = torch.cuda.current_stream().cuda_stream or 1  # 1: the legacy default stream by its own name
    if s["op"] == "qk":
        be.qk_norm_rope(a[0], stream)
        return {"q": s["q_out"], "k": s["k_out"]}
    if s["op"] == "append":
        be.kv8_append(a[0], a[1], a[2], a[3], a[4], stream)
        be.kv8_read(a[0], a[5], a[6], a[7], stream)
        return {"k": s["k_out"], "v": s["v_out"], "scales": s["scales"]}
    be.kv8_attention(a[0], a[1], a[2], a[3], a[4], 0.0, stream)
    return s["out"]


# ---- the plain forms ----------------------------------------------------------------------------------------------
def _rotate(x, cs, rot, half):
    """x [..., hd] in 32 bits rotated by cs [..., rot / 2, 2]: pairs (i, i + rot / 2) or (2 i, 2 i + 1), the rest kept."""
    c, s = cs[..., 0], cs[..., 1]
    a, b = (x[..., :rot // 2], x[..., rot // 2:rot]) if half else (x[..., 0:rot:2], x[..., 1:rot:2])
    u, w = a * c - b * s, a * s + b * c
    y = torch.cat([u, w], -1) if half else torch.stack([u, w], -1).flatten(-2)
    return torch.cat([y, x[..., rot:]], -1)


def _plain_qk(s):
    cs = s["table"][s["positions"].long()][:, None]
    out = {}
    for name in ("q", "k"):
        x, w = s[name].float(), s[name + "_norm"]
        if w is not None:
            x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + 1e-5) * w.float()
        out[name] = _rotate(x, cs, s["rot"], s["half"]).to(s[name].dtype)
    return out


def _index(hd):
    """Where (token, dim) of K and of V lie in a page of one kv head."""
    t, d = torch.arange(PAGE, device="cuda")[:, None], torch.arange(hd, device="cuda")[None]
    return t * hd + (d ^ (64 * (t & 1)) if hd == 128 else d), PAGE * hd + d * PAGE + t


def _places(s, starts, rows):
    """Sequence, position, block and slot of each row of a ragged batch, and whether the row is one (not padding)."""
    r = torch.arange(rows, device="cuda")
    seq = torch.bucketize(r, starts[1:].long(), right=True)
    pos = s["ctx"].long()[seq] - starts[1:].long()[seq] + r
    ok = pos >= 0
    pos = pos.clamp(min=0)
    return seq, pos, s["tables"].long()[seq, pos // PAGE], pos % PAGE, ok


def _plain_append(s):
    hd, rot, pages, scales = s["hd"], s["rot"], s["pages"], s["scales"]
    seq, pos, block, slot, ok = _places(s, s["row_starts"], s["rows"])
    seq, pos, block, slot = seq[ok], pos[ok], block[ok], slot[ok]
    k, v = s["k"][ok].float(), s["v"][ok].float()
    if rot:
        k = _rotate(k, s["table"][pos][:, None], rot, s["half"])
    x = torch.stack([k, v], 2)  # [rows][kv head][side][hd]
    most = torch.zeros_like(scales).index_reduce_(0, block, x.abs().amax(-1), "amax")
    first = torch.full((scales.shape[0],), PAGE, device="cuda").index_reduce_(0, block, slot, "amin")
    old = torch.where((first > 0)[:, None, None], scales, torch.zeros_like(scales))  # a page written from slot 0 is new
    new = torch.maximum(old, most / torch.full_like(most, 127.0))
    touched = torch.nonzero(first < PAGE)[:, 0]
    at = torch.stack(_index(hd))  # [side][token][dim]
    # older tokens of a page whose scale grew: to the new scale
    p = pages[touched]
    q = p[:, :, at].float()  # [pages][kv head][side][token][dim]
    ratio = torch.where(new > 0, old / new, torch.zeros_like(new))[touched]
    kept = (torch.arange(PAGE, device="cuda") < first[touched][:, None])[:, None, None, :, None]
    q = torch.where(kept, torch.round(q * ratio[..., None, None]), q)
    p[:, :, at] = q.to(torch.int8)
    pages[touched] = p
    scale = new[block][..., None]
    q = torch.where(scale > 0, torch.round(x / scale), torch.zeros_like(x)).clamp(-127, 127).to(torch.int8)
    heads = torch.arange(s["kv_heads"], device="cuda")
    for side in range(2):
        pages[block[:, None, None], heads[:, None], at[side][slot][:, None]] = q[:, :, side]
    scales[touched] = new[touched]
    _, _, block, slot, _ = _places(s, s["read_starts"], s["read_rows"])
    got = [(pages[block[:, None, None], heads[:, None], at[i][slot][:, None]].float() * scales[block, :, i, None])
           .to(s["k"].dtype) for i in range(2)]
    return {"k": got[0], "v": got[1], "scales": scales}


def _plain_attend(s):
    hd, h, kvh, n = s["hd"], s["heads"], s["kv_heads"], s["max_rows"]
    seq, pos, _, _, ok = _places(s, s["row_starts"], s["rows"])
    slot = torch.arange(s["rows"], device="cuda") - s["row_starts"].long()[seq]
    q = torch.zeros(s["n"], n, kvh, h // kvh, hd, device="cuda")
    q[seq, slot] = s["q"].float().view(-1, kvh, h // kvh, hd)
    last = torch.full((s["n"], n), -1, device="cuda")
    last[seq, slot] = torch.where(ok, pos, torch.full_like(pos, -1))
    blocks = s["tables"].long()[:, :-(-s["max_ctx"] // PAGE)].clamp(min=0)
    at = _index(hd)
    kv = [(s["pages"][blocks][..., at[i]].float() * s["scales"][blocks][..., i, None, None]).transpose(1, 2).flatten(2, 3)
          for i in range(2)]  # [seq][kv head][token][dim]
    q = q.permute(0, 2, 3, 1, 4).reshape(s["n"], kvh, -1, hd)
    score = torch.matmul(q, kv[0].transpose(-1, -2)).view(s["n"], kvh, h // kvh, n, -1)
    del q
    score *= 1.0 / math.sqrt(hd)
    seen = (torch.arange(score.shape[-1], device="cuda") <= last[..., None])[:, None, None]
    score.masked_fill_(~seen, -math.inf)
    score -= score.amax(-1, keepdim=True).clamp(min=-1e30)
    score.exp_()
    total = score.sum(-1, keepdim=True)
    out = torch.matmul(score.flatten(2, 3), kv[1]).view(s["n"], kvh, h // kvh, n, hd) / total.clamp(min=1e-30)
    return out.permute(0, 3, 1, 2, 4)[seq, slot].reshape(-1, h, hd).to(s["q"].dtype)


# ---- the definition in 64 bits ------------------------------------------------------------------------------------
def _exact_turn(x, table, pos, rot, half):
    """x [rows][heads][hd] times e^(i angle) on its pairs, the angles taken from the table's f32 values."""
    if not rot:
        return x
    w = torch.complex(table[pos, :, 0].double(), table[pos, :, 1].double())[:, None]
    y = x.clone()
    if half:
        z = torch.complex(x[..., :rot // 2].contiguous(), x[..., rot // 2:rot].contiguous()) * w
        y[..., :rot // 2], y[..., rot // 2:rot] = z.real, z.imag
    else:
        z = torch.complex(x[..., 0:rot:2].contiguous(), x[..., 1:rot:2].contiguous()) * w
        y[..., 0:rot:2], y[..., 1:rot:2] = z.real, z.imag
    return y


def exact(c, seed):
    s = prepare(c, seed)
    hd = c["hd"]
    if c["op"] == "qk":
        out = {}
        for name in ("q", "k"):
            x = s[name].double()
            if c["norm"]:
                x = x * (x.pow(2).sum(-1, keepdim=True) / hd + 1e-5).pow(-0.5) * s[name + "_norm"].double()
            out[name] = _exact_turn(x, s["table"], s["positions"].long(), c["rot"], c["half"])
        return out
    lens, kvh = _lens(c), c["kv_heads"]
    pages, scales = s["pages"], s["scales"].double()

    def side(i, b, blocks):
        """[tokens][kv head][dim] whole numbers that the pages of one sequence hold: K (0) or V (1)."""
        p = pages[s["tables"][b, :blocks].long(), :, i * PAGE * hd:(i + 1) * PAGE * hd].double()
        if i:
            p = p.reshape(blocks, kvh, hd, PAGE).permute(0, 3, 1, 2)
        else:
            p = p.reshape(blocks, kvh, PAGE, hd).permute(0, 2, 1, 3).clone()
            if hd == 128:
                p[:, 1::2] = torch.roll(p[:, 1::2], 64, -1)
        return p.reshape(blocks * PAGE, kvh, hd)

    if c["op"] == "append":
        got, r0 = [[], []], 0
        for b, (r, x) in enumerate(lens):
            if x:
                begin = (x - r) // PAGE * PAGE
                ids = s["tables"][b, begin // PAGE:-(-x // PAGE)].long()
                pos = torch.arange(x - r, x, device="cuda")
                new = [_exact_turn(s["k"][r0:r0 + r].double(), s["table"], pos, c["rot"], c["half"]),
                       s["v"][r0:r0 + r].double()]
                for i in range(2):
                    old = side(i, b, -(-x // PAGE))[begin:begin + len(ids) * PAGE].view(-1, PAGE, kvh, hd)
                    rows = torch.zeros(len(ids) * PAGE, kvh, hd, dtype=torch.float64, device="cuda")
                    rows[x - r - begin:x - begin] = new[i]
                    rows = rows.view(-1, PAGE, kvh, hd)
                    before = scales[ids, :, i].clone()
                    before[1 if begin < x - r else 0:] = 0  # only the first page can hold older tokens
                    now = torch.maximum(before, rows.abs().amax((1, 3)) / 127)
                    div = torch.where(now > 0, now, torch.ones_like(now))[:, None, :, None]
                    q = torch.round(rows / div)
                    keep = x - r - begin
                    q[0, :keep] = torch.round(old[0, :keep] * (before[0] / div[0, 0, :, 0])[None, :, None])
                    got[i].append((q * now[:, None, :, None]).view(-1, kvh, hd)[:x - begin])
                    scales[ids, :, i] = now
            r0 += r
        return {"k": torch.cat(got[0]), "v": torch.cat(got[1]), "scales": scales}
    out, r0, group = torch.zeros(s["rows"], c["heads"], hd, dtype=torch.float64, device="cuda"), 0, c["heads"] // kvh
    for b, (r, x) in enumerate(lens):
        if x:
            blocks = -(-x // PAGE)
            ids = s["tables"][b, :blocks].long().repeat_interleave(PAGE)[:x]
            kv = [side(i, b, blocks)[:x] * scales[ids, :, i, None] for i in range(2)]
            seen = torch.ones(r, x, dtype=torch.bool, device="cuda").tril(x - r)
            for h in range(c["heads"]):
                z = s["q"][r0:r0 + r, h].double() @ kv[0][:, h // group].T / hd ** 0.5
                p = torch.softmax(z.masked_fill(~seen, -math.inf), -1)
                out[r0:r0 + r, h] = p @ kv[1][:, h // group]
        r0 += r
    return out
