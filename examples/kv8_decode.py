"""One attention layer over the 8-bit KV cache: ragged prompts in one pass, then decode steps replayed as a CUDA graph.

Every call is one of the framework's: the INT4 projections (ResidentTensor.gemv_device), the norms and the rotation of
q and k (qk_norm_rope), the append into int8 pages (kv8_append) and the attention over them (kv8_attention), with the pages
handed out by BlockManager / BlockTable. torch only owns the buffers. Run on a B200:

    python examples/kv8_decode.py [--steps 32] [--prompts 100 7 33]
"""
from __future__ import annotations

import argparse
import os
import sys

import numpy as np
import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
from paraoxidizer_b200 import _lib as L  # noqa: E402
from paraoxidizer_b200 import quant as Q  # noqa: E402
from paraoxidizer_b200.backend import CudaBackend  # noqa: E402
from paraoxidizer_b200.paged import BlockManager, BlockTable  # noqa: E402

PAGE = 16


class Kv8Layer:
    """qkv and o projections in INT4, norms of q and k, and the 8-bit cache of one layer for up to `seqs` sequences."""

    def __init__(self, be: CudaBackend, hidden=1024, heads=8, kv_heads=2, head_dim=128, seqs=3, most_tokens=512, seed=0):
        rng = np.random.default_rng(seed)
        self.be, self.heads, self.kvh, self.hd, self.hidden = be, heads, kv_heads, head_dim, hidden
        self.w = {}
        for name, rows, cols in (("qkv", (heads + 2 * kv_heads) * head_dim, hidden), ("o", hidden, heads * head_dim)):
            w = rng.standard_normal(rows * cols, dtype=np.float32) * np.float32(0.5 / cols ** 0.5)
            packed, scales = Q.quantize_int4_group(w, 128)
            self.w[name] = be.upload_int4(packed, scales, rows, cols, 128)
        norm = lambda: torch.from_numpy((1 + 0.1 * rng.standard_normal(head_dim)).astype(np.float16)).cuda()  # noqa: E731
        self.q_norm, self.k_norm = norm(), norm()
        inv = 500000.0 ** (-np.arange(0, head_dim, 2) / head_dim)
        ang = np.arange(most_tokens)[:, None] * inv
        self.table = torch.from_numpy(np.stack([np.cos(ang), np.sin(ang)], -1).astype(np.float32)).cuda()
        self.rope = L.Rope(self.table.data_ptr(), most_tokens, head_dim, L.POX_ROPE_INTERLEAVED)
        # the cache: pages of 16 tokens, a scale for each page, kv head and side
        self.width = most_tokens // PAGE
        blocks = seqs * self.width
        self.manager, self.tables = BlockManager(blocks), [BlockTable() for _ in range(seqs)]
        self.pages = torch.empty(blocks, kv_heads, 32 * head_dim, dtype=torch.int8, device="cuda")
        self.scales = torch.empty(blocks, kv_heads, 2, device="cuda")
        self.cache = L.Kv8Cache(self.pages.data_ptr(), self.scales.data_ptr(), blocks, kv_heads, head_dim)
        self.block_tables = torch.full((seqs, self.width), -1, dtype=torch.int32, device="cuda")
        self.ctx = torch.zeros(seqs, dtype=torch.int32, device="cuda")

    def reserve(self, tokens):
        """Pages for tokens[s] more tokens of each sequence."""
        for s, n in enumerate(tokens):
            self.tables[s].reserve(self.manager, n)
            self.tables[s].sequence_len += n
            self.block_tables[s].copy_(torch.from_numpy(self.tables[s].as_array(self.width)))

    def buffers(self, rows):
        z = lambda n: torch.empty(rows, n, device="cuda")  # noqa: E731
        return dict(qkv=z((self.heads + 2 * self.kvh) * self.hd), att=z(self.heads * self.hd), out=z(self.hidden),
                    x=z(self.hidden), pos=torch.zeros(rows, dtype=torch.int32, device="cuda"))

    def forward(self, b, row_starts, max_rows, stream):
        """b['x'] -> b['out'] for rows whose positions are b['pos']; the sequences' contexts (new rows included) are self.ctx."""
        rows, hd, h, kvh = b["x"].shape[0], self.hd, self.heads, self.kvh
        ld, at = (h + 2 * kvh) * hd, b["qkv"].data_ptr()
        q, k, v = (L.Rows(at + 4 * hd * o, L.POX_F32, ld, hd) for o in (0, h, h + kvh))
        batch = L.Kv8Batch(row_starts.data_ptr() if row_starts is not None else 0, self.ctx.data_ptr(),
                           self.block_tables.data_ptr(), self.ctx.shape[0], rows, max_rows, self.width * PAGE, self.width)
        self.w["qkv"].gemv_device(b["x"].data_ptr(), rows, at, stream)
        self.be.qk_norm_rope(L.QkNormRope(q, k, q, k, rows, h, kvh, hd, self.q_norm.data_ptr(), self.k_norm.data_ptr(), 1e-5,
                                          self.rope, b["pos"].data_ptr()), stream)
        self.be.kv8_append(self.cache, batch, k, v, None, stream)  # (k is rotated already)
        self.be.kv8_attention(self.cache, batch, q, L.Rows(b["att"].data_ptr(), L.POX_F32, h * hd, hd), h, 0.0, stream)
        self.w["o"].gemv_device(b["att"].data_ptr(), rows, b["out"].data_ptr(), stream)


def run(prompts=(100, 7, 33), steps=32, seed=0):
    """Prompts of those lengths, then `steps` tokens of each sequence (the layer's output fed back as the next input).
    Returns (outputs of the prompts' rows, outputs of the steps [steps][seqs][hidden], microseconds a step, the layer)."""
    be = CudaBackend.create(0)
    layer = Kv8Layer(be, seqs=len(prompts), seed=seed)
    st = torch.cuda.Stream()
    with torch.cuda.stream(st):
        g = torch.Generator(device="cuda").manual_seed(seed)
        rows = sum(prompts)
        b = layer.buffers(rows)
        b["x"].normal_(generator=g)
        starts = torch.tensor(np.concatenate([[0], np.cumsum(prompts)]), dtype=torch.int32, device="cuda")
        b["pos"].copy_(torch.cat([torch.arange(n) for n in prompts]))
        layer.reserve([n + steps for n in prompts])
        layer.ctx.copy_(torch.tensor(prompts))
        layer.forward(b, starts, max(prompts), st.cuda_stream)

        d = layer.buffers(len(prompts))
        d["x"].copy_(b["out"][starts[1:].long() - 1])
        d["pos"].copy_(layer.ctx - 1)
        outs = torch.empty(steps, len(prompts), layer.hidden, device="cuda")
        at = torch.zeros(1, dtype=torch.long, device="cuda")

        def step():
            layer.ctx.add_(1)
            d["pos"].add_(1)
            layer.forward(d, None, 1, st.cuda_stream)
            d["x"].copy_(torch.nn.functional.normalize(d["out"]) * layer.hidden ** 0.5)
            outs.index_copy_(0, at, d["out"][None])
            at.add_(1)

        step()  # sizes every buffer before the capture
        graph = torch.cuda.CUDAGraph()
        st.synchronize()
        with torch.cuda.graph(graph, stream=st):
            step()
        t0, t1 = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        t0.record()
        for _ in range(steps - 1):
            graph.replay()
        t1.record()
    be.synchronize()  # reports what a kernel found wrong with its input
    return b["out"], outs, t0.elapsed_time(t1) * 1e3 / max(1, steps - 1), layer


if __name__ == "__main__":
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--prompts", type=int, nargs="+", default=[100, 7, 33])
    ap.add_argument("--steps", type=int, default=32)
    a = ap.parse_args()
    _, outs, us, layer = run(tuple(a.prompts), a.steps)
    held = layer.pages.numel() + 4 * layer.scales.numel()
    print(f"{len(a.prompts)} sequences, {a.steps} steps: {us:.1f} us a step (one layer), output rms "
          f"{float(outs.pow(2).mean().sqrt()):.4f}, cache {held / 2**20:.2f} MiB "
          f"(f16 pages: {2 * layer.pages.numel() / 2**20:.2f} MiB)")
