"""A decoder layer that answers in low bits: MXFP4 weights and activations in its seven
products, keys and values in the paged 8-bit cache, attention over the codes.

    python examples/low_bit_layer.py

runs a Qwen3-0.6B-shaped layer on ragged prompts, then token by token, and prints how far its
outputs are from the same layer in float32 and what a step takes.
"""
import os
import sys
import time

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

from perm_amd import kvcache, mxfp4  # noqa: E402
from perm_amd.workloads import QWEN3_06B_DIMS, qwen3_layer_weights  # noqa: E402


def rms_norm(x):
    return x * torch.rsqrt(x.float().square().mean(-1, keepdim=True) + 1e-6).to(x.dtype)


def rotate(x, pos, base=1e6):
    """Rotary positions, half layout: x [rows, heads, d], pos [rows]."""
    half = x.shape[-1] // 2
    freq = base ** (-torch.arange(half, device=x.device) / half)
    angle = (pos[:, None] * freq)[:, None]
    a, b = x[..., :half].float(), x[..., half:].float()
    cos, sin = angle.cos(), angle.sin()
    return torch.cat([a * cos - b * sin, b * cos + a * sin], -1).to(x.dtype)


class LowBitLayer:
    """The layer's weights in MXFP4. ``forward`` takes the rows of a ragged batch and the cache
    they are appended to; the caller keeps the cache, its page table and the lengths."""

    def __init__(self, weights, dims):
        self.w = {name: mxfp4.quantize(w) for name, w in weights.items()}
        self.heads, self.kv_heads, self.d = dims["n_heads"], dims["n_kv"], dims["head_dim"]

    def forward(self, x, pos, cache, table, filled, lens, offsets=None):
        h = rms_norm(x)
        rows = x.shape[0]
        q = mxfp4.linear(h, self.w["attn_q"]).view(rows, self.heads, self.d)
        k = mxfp4.linear(h, self.w["attn_k"]).view(rows, self.kv_heads, self.d)
        v = mxfp4.linear(h, self.w["attn_v"]).view(rows, self.kv_heads, self.d)
        kvcache.write(cache, rotate(k, pos), v, table, filled, offsets)
        o = kvcache.attention(rotate(q, pos), cache, table, lens, offsets)
        x = x + mxfp4.linear(o.reshape(rows, -1), self.w["attn_output"])
        h = rms_norm(x)
        gate = mxfp4.linear(h, self.w["ffn_gate"])
        up = mxfp4.linear(h, self.w["ffn_up"])
        return x + mxfp4.linear(torch.nn.functional.silu(gate) * up, self.w["ffn_down"])


def float_layer(weights, dims, x):
    """The same layer in float32 on one whole sequence x [n, d_model]."""
    w = {n: t.float() for n, t in weights.items()}
    n, d = x.shape[0], dims["head_dim"]
    pos = torch.arange(n, device=x.device)
    h = rms_norm(x)
    q = rotate((h @ w["attn_q"].t()).view(n, -1, d), pos).transpose(0, 1)
    k = rotate((h @ w["attn_k"].t()).view(n, -1, d), pos).transpose(0, 1)
    v = (h @ w["attn_v"].t()).view(n, -1, d).transpose(0, 1)
    group = q.shape[0] // k.shape[0]
    k, v = k.repeat_interleave(group, 0), v.repeat_interleave(group, 0)
    s = (q @ k.transpose(1, 2).contiguous()) * d ** -0.5
    s = s.masked_fill(pos[None, :] > pos[:, None], float("-inf"))
    o = (torch.softmax(s, -1) @ v).transpose(0, 1).reshape(n, -1)
    x = x + o @ w["attn_output"].t()
    h = rms_norm(x)
    return x + (torch.nn.functional.silu(h @ w["ffn_gate"].t()) * (h @ w["ffn_up"].t())) @ w["ffn_down"].t()


def run(prompts=(37, 200, 5, 91), steps=8, block=16, seed=0):
    """Prompts of these lengths, then ``steps`` tokens of each; {"prompt": relative error of the
    prompts' rows, "tokens": of the generated rows, "ms_per_token": ...}."""
    dims = QWEN3_06B_DIMS
    weights = qwen3_layer_weights(0, seed)
    layer = LowBitLayer(weights, dims)
    g = torch.Generator(device="cuda")
    g.manual_seed(seed + 1)
    seqs = [torch.randn((n + steps, dims["d_model"]), generator=g, device="cuda") for n in prompts]
    want = [float_layer(weights, dims, x) for x in seqs]

    batch, cap = len(prompts), -(-(max(prompts) + steps) // block)
    cache = kvcache.new(batch * cap, dims["n_kv"], dims["head_dim"], block)
    table = torch.randperm(batch * cap, generator=g, device="cuda").view(batch, cap).to(torch.int32)
    i32 = dict(dtype=torch.int32, device="cuda")
    lens = torch.tensor(prompts, **i32)
    offsets = torch.tensor([sum(prompts[:i]) for i in range(batch + 1)], **i32)
    pos = torch.cat([torch.arange(n, device="cuda") for n in prompts])
    x = torch.cat([s[:n] for s, n in zip(seqs, prompts)]).to(torch.bfloat16)
    y = layer.forward(x, pos, cache, table, torch.zeros_like(lens), lens, offsets)
    ref = torch.cat([w[:n] for w, n in zip(want, prompts)])
    out = {"prompt": float((y.float() - ref).norm() / ref.norm())}

    err = norm = 0.0
    torch.cuda.synchronize()
    spent = 0.0
    for t in range(steps):
        x = torch.stack([s[n + t] for s, n in zip(seqs, prompts)]).to(torch.bfloat16)
        torch.cuda.synchronize()
        began = time.perf_counter()
        y = layer.forward(x, lens, cache, table, lens, lens + 1)
        torch.cuda.synchronize()
        spent += time.perf_counter() - began
        lens = lens + 1
        ref = torch.stack([w[n + t] for w, n in zip(want, prompts)])
        err += float((y.float() - ref).square().sum())
        norm += float(ref.square().sum())
    out["tokens"] = (err / norm) ** 0.5
    out["ms_per_token"] = 1e3 * spent / steps
    return out


if __name__ == "__main__":
    got = run()
    print(f"relative error against float32: prompts {got['prompt']:.4f}, tokens {got['tokens']:.4f}; "
          f"{got['ms_per_token']:.2f} ms a step of four sequences")
