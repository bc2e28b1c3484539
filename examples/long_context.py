"""The attention half of a decoder layer over contexts that outgrow the cache, from the operators of castforge_amd.ops:

  norm, as E4M3 codes  ->  block-scaled FP8 product (queries, keys, values)  ->  rotation and append to the paged 8-bit cache
  ->  attention, which adds up the weights that each cached token gets  ->  FP8 product

After the prompt, and whenever a sequence's pages are full, the tokens of greatest weight, the first ones and the last ones move
to other pages, and the step goes on with those.  The step is captured in a HIP graph once and replayed.
`python examples/long_context.py` prints the outputs' distance from the same layer in float32 over all tokens, the time of a
step and that of an eviction."""
import argparse
import sys
import time
from pathlib import Path

import torch

sys.path[:0] = [str(Path(__file__).resolve().parent.parent), str(Path(__file__).resolve().parent)]
from castforge_amd import ops  # noqa: E402
from decoder_attention import AttentionHalf, distance  # noqa: E402


class Pages:
    """Two sets of pages a sequence, `cols` each, behind the `prompt_cols` that its prompt is read into: an eviction reads the one and
    fills the other."""

    def __init__(self, batch: int, prompt_cols: int, cols: int, seed: int = 0):
        g = torch.Generator(device="cuda").manual_seed(seed)
        self.num = batch * (prompt_cols + 2 * cols)
        all_pages = torch.randperm(self.num, generator=g, device="cuda").int().view(batch, -1)
        self.prompt, a, b = (t.contiguous() for t in all_pages.split((prompt_cols, cols, cols), 1))
        self.sets = [a, b]

    def spare(self):
        """The set that is not in use, which is in use from now on."""
        self.sets.reverse()
        return self.sets[0]


class Decoder:
    """Sequences whose prompts are read: the layer, their pages, lengths and the weights that their tokens got."""

    def __init__(self, layer, prompts, x, budget: int, room: int, sinks: int, recent: int, page: int, seed: int = 0):
        self.layer, self.budget, self.room, self.sinks, self.recent = layer, budget, room, sinks, recent
        batch, dev = len(prompts), "cuda"
        self.pages = Pages(batch, -(-max(prompts) // page), -(-(budget + room) // page), seed)
        self.cache = ops.Kv8Cache.empty(self.pages.num, layer.kv_heads, page, layer.head_dim, device=dev)
        self.kv_lens = torch.tensor(prompts, dtype=torch.int32, device=dev)
        self.positions = torch.tensor(prompts, device=dev)
        positions = torch.cat([torch.arange(n, device=dev) for n in prompts])
        cu = torch.nn.functional.pad(self.kv_lens.cumsum(0), (1, 0)).int()
        weights = torch.zeros((batch, layer.kv_heads, max(prompts)), device=dev)
        self.prompt_out = self.half(torch.cat([t[:n] for t, n in zip(x, prompts)]), positions, self.pages.prompt, self.kv_lens, weights, cu)
        self.table = self.pages.sets[0].clone()
        self.weights = torch.zeros((batch, layer.kv_heads, budget + room), device=dev)
        self.cut(self.pages.prompt, weights)

    def half(self, x, positions, table, kv_lens, weights, cu_q=None):
        layer = self.layer
        codes, scales, _ = ops.rms_norm_fp8(x, layer.norm, block=128)
        rows = ops.gemm_fp8_block(codes, scales, *layer.qkv).unflatten(1, (-1, layer.head_dim))
        q, k, v = rows.split((layer.q_heads, layer.kv_heads, layer.kv_heads), 1)
        q = ops.kv8_append(self.cache, k, v, table, kv_lens, cu_q=cu_q, positions=positions, cos=layer.cos, sin=layer.sin, q=q)
        o = ops.kv8_attention(q, self.cache, table, kv_lens, cu_q=cu_q, weights=weights)
        return ops.gemm_fp8_block(*ops.quantize_fp8_block(o.flatten(1)), *layer.out)

    def cut(self, table, weights):
        """To the budget, in the other set of pages."""
        new = self.pages.spare()
        _, lens, kept = ops.kv8_evict(self.cache, table, self.kv_lens, weights, self.budget, new, sinks=self.sinks, recent=self.recent)
        self.table.copy_(new), self.kv_lens.copy_(lens)
        self.weights.zero_()
        self.weights[..., :self.budget] = kept
        self.most = self.budget  # tokens a sequence, at most

    def before_step(self):
        """Makes room for a token of each sequence, and counts it."""
        if self.most == self.budget + self.room:
            self.cut(self.table, self.weights)
        self.most += 1
        self.kv_lens += 1

    def step(self, x):
        return self.half(x, self.positions, self.table, self.kv_lens, self.weights)


def run(prompts=(3000, 500, 20), new_tokens=80, budget=512, room=32, sinks=4, recent=64, hidden=1024, q_heads=8, kv_heads=2, head_dim=128,
        page=16, seed=0):
    """Prompts, then new_tokens single tokens of each sequence, by plain calls and by replay.  Returns the outputs of the single tokens
    of both ways and of float32 over all tokens, [sequence][token], and the seconds of a replayed step and of an eviction."""
    layer, dev, batch = AttentionHalf(hidden, q_heads, kv_heads, head_dim, seed=seed), "cuda", len(prompts)
    g = torch.Generator(device=dev).manual_seed(seed + 1)
    total = [n + new_tokens for n in prompts]
    x = [torch.randn((n, hidden), generator=g, device=dev).bfloat16() for n in total]

    def new_decoder():
        return Decoder(layer, list(prompts), x, budget, room, sinks, recent, page, seed)

    def rows(i):
        return torch.stack([t[n + i] for t, n in zip(x, prompts)])

    one, called = new_decoder(), []
    for i in range(new_tokens):
        one.before_step()
        called.append(one.step(rows(i)))
        one.positions += 1

    one, replayed = new_decoder(), []
    static = rows(0)
    warm = new_decoder()  # loads the kernels
    warm.before_step()
    warm.step(static)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = one.step(static)
    for i in range(new_tokens):
        one.before_step()
        static.copy_(rows(i))
        graph.replay()
        replayed.append(y.clone())
        one.positions += 1

    times = []
    for work in (graph.replay, lambda: ops.kv8_evict(one.cache, one.table, one.kv_lens, one.weights, budget, one.pages.sets[1], sinks=sinks, recent=recent)):
        work()
        torch.cuda.synchronize()
        start = time.perf_counter()
        for _ in range(100):
            work()
        torch.cuda.synchronize()
        times.append((time.perf_counter() - start) / 100)
    nothing = torch.zeros((sum(total), hidden), device=dev)
    plain = layer.plain(torch.cat(x), nothing, total).split(total)
    return torch.stack(called, 1).unbind(), torch.stack(replayed, 1).unbind(), [t[n:] for t, n in zip(plain, prompts)], times


if __name__ == "__main__":
    args = argparse.ArgumentParser()
    for name, value in (("hidden", 4096), ("q-heads", 32), ("kv-heads", 8), ("head-dim", 128), ("tokens", 200), ("budget", 1024), ("room", 64)):
        args.add_argument("--" + name, type=int, default=value)
    args.add_argument("--prompts", type=int, nargs="+", default=[4000, 1000, 64])
    a = args.parse_args()
    called, replayed, plain, (step, evict) = run(a.prompts, a.tokens, a.budget, a.room, hidden=a.hidden, q_heads=a.q_heads, kv_heads=a.kv_heads,
                                                 head_dim=a.head_dim)
    print(f"distance from float32 over all tokens: {distance(called, plain):.3f} by calls, {distance(replayed, plain):.3f} by replay; "
          f"{1e6 * step:.1f} us a replayed step of {len(a.prompts)} sequences, {1e6 * evict:.1f} us an eviction")
