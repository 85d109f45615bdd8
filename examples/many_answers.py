"""Several answers to each of some prompts from one cache: the prompts' pages are shared, read once for
all of their answers, and every answer's next token is drawn with settings of its own.

    python examples/many_answers.py

runs two Qwen3-0.6B-shaped layers in low bits (``low_bit_layer``) under a random output matrix, and
prints what a step takes and how many pages the answers hold, beside what they would without sharing.
"""
import os
import sys
import time

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))

from low_bit_layer import LowBitLayer, rms_norm, rotate  # noqa: E402
from perm_amd import kvcache, kvpages, mxfp4, sampling  # noqa: E402
from perm_amd.workloads import QWEN3_06B_DIMS, qwen3_layer_weights  # noqa: E402


class SharedLayer(LowBitLayer):
    """The layer over sequences that begin alike: ``shared`` pages of every group's."""

    def forward(self, x, pos, cache, table, filled, lens, offsets=None, shared=None):
        h = rms_norm(x)
        rows = x.shape[0]
        q = mxfp4.linear(h, self.w["attn_q"]).view(rows, self.heads, self.d)
        k = mxfp4.linear(h, self.w["attn_k"]).view(rows, self.kv_heads, self.d)
        v = mxfp4.linear(h, self.w["attn_v"]).view(rows, self.kv_heads, self.d)
        kvcache.write(cache, rotate(k, pos), v, table, filled, offsets)
        o = kvcache.attention(rotate(q, pos), cache, table, lens, offsets, shared=shared)
        x = x + mxfp4.linear(o.reshape(rows, -1), self.w["attn_output"])
        h = rms_norm(x)
        gate, up = mxfp4.linear(h, self.w["ffn_gate"]), mxfp4.linear(h, self.w["ffn_up"])
        return x + mxfp4.linear(torch.nn.functional.silu(gate) * up, self.w["ffn_down"])


def run(prompts=(300, 170), answers=8, steps=24, layers=2, vocab=1000, block=16, seed=0):
    """{"tokens": [sequences, steps], "pages": held at the end, "alone": what the sequences' pages would be
    without sharing, "ms_per_token": ...}. A group is a prompt's row of the table and its answers'."""
    dims = QWEN3_06B_DIMS
    stack = [SharedLayer(qwen3_layer_weights(i, seed), dims) for i in range(layers)]
    g = torch.Generator(device="cuda").manual_seed(seed)
    embed = torch.randn((vocab, dims["d_model"]), generator=g, device="cuda").to(torch.bfloat16)
    head = mxfp4.quantize(torch.randn((vocab, dims["d_model"]), generator=g, device="cuda") * 0.1)
    i32 = dict(dtype=torch.int32, device="cuda")

    groups, batch = len(prompts), len(prompts) * answers
    cap = -(-(max(prompts) + steps) // block)
    pages = sum(-(-n // block) for n in prompts) + batch * (-(-steps // block) + 2)
    caches = [kvcache.new(pages, dims["n_kv"], dims["head_dim"], block) for _ in stack]
    refs, table = kvpages.new(pages), torch.full((batch, cap), -1, **i32)

    # the prompts, in the first row of each group
    zero = torch.zeros(batch, **i32)
    counts = [prompts[i // answers] if i % answers == 0 else 0 for i in range(batch)]
    lens = torch.tensor(counts, **i32)
    offsets = torch.tensor([sum(counts[:i]) for i in range(batch + 1)], **i32)
    _, _, missing = kvpages.grow(refs, table, zero, lens, block)
    pos = torch.cat([torch.arange(n, device="cuda") for n in prompts])
    x = embed[torch.randint(0, vocab, (sum(prompts),), generator=g, device="cuda")]
    for layer, cache in zip(stack, caches):
        x = layer.forward(x, pos, cache, table, zero, lens, offsets)
    last = x[offsets[1::answers].long() - 1].repeat_interleave(answers, 0)

    # the answers
    first = torch.arange(0, batch, answers, **i32)
    children = torch.tensor([i for i in range(batch) if i % answers], **i32)
    kvpages.fork(refs, table, lens, first.repeat_interleave(answers - 1), children, block)
    lens = torch.tensor([n for n in prompts for _ in range(answers)], **i32)
    shared = torch.tensor([n // block for n in prompts], **i32)
    settings = dict(temperature=torch.linspace(0.6, 1.2, batch, device="cuda"), top_k=50, top_p=0.95)
    out, x = [], last
    torch.cuda.synchronize()
    began = time.perf_counter()
    for _ in range(steps):
        u = torch.rand(batch, generator=g, device="cuda")
        token = sampling.sample(mxfp4.linear(rms_norm(x), head, torch.float32), u, **settings)
        out.append(token)
        src, dst, more = kvpages.grow(refs, table, lens, 1, block)
        missing = missing + more
        x = embed[token.long()]
        for layer, cache in zip(stack, caches):
            kvpages.copy(cache, src, dst)
            x = layer.forward(x, lens, cache, table, lens, lens + 1, shared=shared)
        lens = lens + 1
    torch.cuda.synchronize()
    spent = time.perf_counter() - began
    if int(missing.sum()):
        raise RuntimeError("the cache has too few pages")
    return {"tokens": torch.stack(out, 1), "pages": int((refs > 0).sum()),
            "alone": sum(-(-int(n) // block) for n in lens), "groups": groups,
            "ms_per_token": 1e3 * spent / steps}


if __name__ == "__main__":
    got = run()
    print(f"{got['tokens'].shape[0]} answers hold {got['pages']} pages, {got['alone']} without sharing; "
          f"{got['ms_per_token']:.2f} ms a step")
