"""The 8-bit cache in use: several sequences' prompts, then single tokens.

Each layer rotates its queries and keys by positions with three axes (time,
height, width), writes keys and values into the 8-bit cache and attends over
it.  The prompts have different lengths and go through in one batch; the
token steps after them are one CUDA graph, replayed with the sequences' new
lengths.  The layers' projections are random matrices: the example shows the
calls and their order, not a trained model.

    python shannon-prime-llama_b200/examples/q8_layers.py [--layers 4] [--steps 16]
"""
from __future__ import annotations

import argparse
import math
import sys
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parent.parent))
import spb200  # noqa: E402


class Layers:
    """A stack of attention layers over one 8-bit cache."""

    def __init__(self, n_layers: int, n_q_heads: int, n_kv_heads: int, head_dim: int, n_seqs: int, max_seq_len: int,
                 stream, fmt: str = "e4m3", block_tokens: int = 64, seed: int = 0):
        g = torch.Generator(device="cuda").manual_seed(seed)
        self.hq, self.hk, self.hd = n_q_heads, n_kv_heads, head_dim
        width = n_q_heads * head_dim
        self.width = width
        self.qkv = [torch.randn(width, (n_q_heads + 2 * n_kv_heads) * head_dim, generator=g, device="cuda",
                                dtype=torch.float16) / math.sqrt(width) for _ in range(n_layers)]
        self.o = [torch.randn(width, width, generator=g, device="cuda", dtype=torch.float16) / math.sqrt(width)
                  for _ in range(n_layers)]
        pairs = head_dim // 2
        self.rope = spb200.RopeAxes(head_dim, [pairs - 2 * (3 * pairs // 8), 3 * pairs // 8, 3 * pairs // 8], pairing="halves")
        self.stream = stream                    # everything runs on this one
        self.cache = spb200.Q8Cache(head_dim, n_layers, n_kv_heads, max_seq_len, n_seqs=n_seqs, fmt=fmt,
                                    block_tokens=block_tokens, stream=stream)

    def __call__(self, x, pos, batch):
        """x [tokens][width] fp16, pos int32 [3][tokens]."""
        n = x.shape[0]
        for layer, (wqkv, wo) in enumerate(zip(self.qkv, self.o)):
            qkv = (x @ wqkv).view(n, self.hq + 2 * self.hk, self.hd)
            q, k, v = qkv.split([self.hq, self.hk, self.hk], 1)
            self.rope.apply(pos, q, k, q_out=q, k_out=k, stream=self.stream)  # in place, in the projection's rows
            self.cache.write_kv_tokens(layer, batch, k, v)
            y = self.cache.attn(layer, batch, q, logit_scale=1.0 / math.sqrt(self.hd), stream=self.stream)
            x = x + y.view(n, self.width) @ wo
        return x


def main(argv=None) -> float:
    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    ap.add_argument("--layers", type=int, default=4)
    ap.add_argument("--steps", type=int, default=16)
    ap.add_argument("--fmt", choices=("int8", "e4m3"), default="e4m3")
    a = ap.parse_args(argv)
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        return run(a, stream)


def run(a, stream) -> float:
    lens = [77, 1024, 3, 350]
    most = max(lens) + a.steps
    net = Layers(a.layers, 16, 4, 128, len(lens), most, stream, fmt=a.fmt)
    scale = 1.0 / math.sqrt(net.hd)
    g = torch.Generator(device="cuda").manual_seed(1)

    # ---- the prompts, packed
    cu = torch.tensor([0, *torch.tensor(lens).cumsum(0).tolist()], dtype=torch.int32, device="cuda")
    kv = torch.tensor(lens, dtype=torch.int32, device="cuda")
    x = torch.randn(sum(lens), net.width, generator=g, device="cuda", dtype=torch.float16)
    t = torch.cat([torch.arange(n) for n in lens])
    pos = torch.stack([t // 64, t % 64 // 8, t % 8]).to(dtype=torch.int32, device="cuda").contiguous()   # frames of 8 x 8
    y = net(x, pos, spb200.Q8Batch(cu, kv, sum(lens), max(lens), max(lens)))

    # ---- single tokens: a step's calls captured once, replayed with other lengths and positions
    n = len(lens)
    batch = spb200.Q8Batch(torch.arange(n + 1, dtype=torch.int32, device="cuda"), kv, n, 1, most)
    x1 = y[(cu[1:] - 1).long()]
    p1 = torch.empty(3, n, dtype=torch.int32, device="cuda")

    def step():
        kv.add_(1)
        p1.copy_((kv - 1).expand(3, n))
        y = net(x1, p1, batch)
        x1.copy_(y * (math.sqrt(net.width) / y.float().norm(dim=-1, keepdim=True)).half())

    step()                                      # the first as it is: workspaces and libraries get ready
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        step()
    for _ in range(a.steps - 1):
        graph.replay()
    if net.cache.status(stream=stream):
        raise RuntimeError("the cache reported an error")

    # ---- attention of layer 0 against the formula over the keys and values read back
    q = torch.randn(n, net.hq, net.hd, generator=g, device="cuda", dtype=torch.float16)
    got = net.cache.attn(0, batch, q, logit_scale=scale, stream=stream).double()
    off = 0.0
    for s, length in enumerate(kv.tolist()):
        kv_back = torch.empty(2, length, net.hk, net.hd, device="cuda")
        for which in (0, 1):
            net.cache.read_kv_tokens(which, 0, s, 0, kv_back[which])
        k, v = kv_back.double().repeat_interleave(net.hq // net.hk, 2)
        w = torch.softmax(torch.einsum("hd,thd->ht", q[s].double(), k) * scale, -1)
        want = torch.einsum("ht,thd->hd", w, v)
        off = max(off, ((got[s] - want).norm() / want.norm()).item())
    print(f"{a.layers} layers, prompts of {lens} tokens, {a.steps} single-token steps in a graph: "
          f"attention within {off:.1e} of the values read back")
    return off


if __name__ == "__main__":
    sys.exit(0 if main() < 2e-3 else 1)
