"""The attention half of a decoder layer, a prompt and then single tokens, from the operators of castforge_amd.ops:

  norm of the residual's sum, as E4M3 codes  ->  block-scaled FP8 product (queries, keys, values)
  ->  rotation and append to the paged 4-bit cache  ->  attention over the cache  ->  FP8 product  ->  the next residual

The step of single tokens is captured in a HIP graph once and replayed: between tokens only the small index tensors
change.  `python examples/decoder_attention.py` prints the outputs' distance from the same layer in float32 and the
time of a step."""
import argparse
import sys
import time
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parent.parent))
from castforge_amd import ops  # noqa: E402


class AttentionHalf:
    """Weights of one layer: a norm, the joint projection to queries, keys and values, and the output's projection."""

    def __init__(self, hidden: int, q_heads: int, kv_heads: int, head_dim: int, max_pos: int = 8192, seed: int = 0):
        g = torch.Generator(device="cuda").manual_seed(seed)
        self.q_heads, self.kv_heads, self.head_dim = q_heads, kv_heads, head_dim
        self.norm = (1 + 0.1 * torch.randn(hidden, generator=g, device="cuda")).bfloat16()
        self.w_qkv = torch.randn(((q_heads + 2 * kv_heads) * head_dim, hidden), generator=g, device="cuda") * hidden ** -0.5
        self.w_out = torch.randn((hidden, q_heads * head_dim), generator=g, device="cuda") * (q_heads * head_dim) ** -0.5
        self.qkv, self.out = (ops.quantize_fp8_block(w, block_rows=128) for w in (self.w_qkv, self.w_out))
        half = head_dim // 2
        angle = torch.arange(max_pos, device="cuda")[:, None] * 10000.0 ** (-torch.arange(half, device="cuda") / half)
        self.cos, self.sin = angle.cos(), angle.sin()

    def __call__(self, x, residual, cache, slots, positions, table, kv_lens, cu_q=None):
        """x and residual bf16 [T, hidden]; returns the layer's output and the residual's sum."""
        codes, scales, h = ops.rms_norm_fp8(x, self.norm, residual=residual, block=128)
        rows = ops.gemm_fp8_block(codes, scales, *self.qkv).unflatten(1, (-1, self.head_dim))
        q, k, v = rows.split((self.q_heads, self.kv_heads, self.kv_heads), 1)  # slices: no copies
        q = ops.kv4_append(cache, k, v, slots, positions, self.cos, self.sin, q=q)
        o = ops.kv4_attention(q, cache, table, kv_lens, cu_q=cu_q)
        return ops.gemm_fp8_block(*ops.quantize_fp8_block(o.flatten(1)), *self.out), h

    def plain(self, x, residual, lens):
        """The same in float32, whole sequences at once."""
        h = (x.float() + residual.float())
        y = h * torch.rsqrt(h.square().mean(1, keepdim=True) + 1e-6) * self.norm.float()
        outs, half, ratio = [], self.head_dim // 2, self.q_heads // self.kv_heads
        for rows in (y @ self.w_qkv.t()).unflatten(1, (-1, self.head_dim)).split(lens):
            q, k, v = rows.split((self.q_heads, self.kv_heads, self.kv_heads), 1)
            c, s = self.cos[:len(rows), None], self.sin[:len(rows), None]
            q, k = (torch.cat([t[..., :half] * c - t[..., half:] * s, t[..., half:] * c + t[..., :half] * s], -1) for t in (q, k))
            k, v = (t.repeat_interleave(ratio, 1) for t in (k, v))
            scores = torch.matmul(q.transpose(0, 1), k.transpose(0, 1).transpose(1, 2).contiguous()) * self.head_dim ** -0.5
            scores += torch.full(scores.shape[1:], -torch.inf, device=x.device).triu(1)
            outs.append(torch.matmul(scores.softmax(-1), v.transpose(0, 1).contiguous()).transpose(0, 1).flatten(1))
        return torch.cat(outs) @ self.w_out.t()


def run(prompts=(300, 17, 1), new_tokens=8, hidden=1024, q_heads=8, kv_heads=2, head_dim=128, page=16, seed=0):
    """Prompts of the given lengths, then new_tokens single tokens of each sequence, by replay and by plain calls.  Returns the
    outputs of both ways and of float32, all [sequence][token]."""
    layer, batch, dev = AttentionHalf(hidden, q_heads, kv_heads, head_dim, seed=seed), len(prompts), "cuda"
    g = torch.Generator(device=dev).manual_seed(seed + 1)
    total = [n + new_tokens for n in prompts]
    x, res = ([torch.randn((n, hidden), generator=g, device=dev).bfloat16() for n in total] for _ in range(2))

    # pages of a sequence lie anywhere in the cache
    cols = -(-max(total) // page)
    pages = torch.randperm(batch * cols, generator=g, device=dev).view(batch, cols)
    table = pages.int()

    def slots_of(seq, positions):
        return pages[seq, positions // page] * page + positions % page

    def prompt(cache):
        seq = torch.repeat_interleave(torch.arange(batch, device=dev), torch.tensor(prompts, device=dev))
        pos = torch.cat([torch.arange(n, device=dev) for n in prompts])
        lens = torch.tensor(prompts, dtype=torch.int32, device=dev)
        cu = torch.nn.functional.pad(lens.cumsum(0), (1, 0)).int()
        rows = (torch.cat([t[:n] for t, n in zip(v, prompts)]) for v in (x, res))
        return layer(*rows, cache, slots_of(seq, pos), pos, table, lens, cu_q=cu)[0].split(list(prompts))

    def new_cache():
        return ops.Kv4Cache.empty(batch * cols, kv_heads, page, head_dim, group=head_dim, device=dev)

    # single tokens, call by call
    cache, seq = new_cache(), torch.arange(batch, device=dev)
    called = [list(t.unbind()) for t in prompt(cache)]
    for i in range(new_tokens):
        pos = torch.tensor([n + i for n in prompts], device=dev)
        rows = (torch.stack([t[n + i] for t, n in zip(v, prompts)]) for v in (x, res))
        y = layer(*rows, cache, slots_of(seq, pos), pos, table, (pos + 1).int())[0]
        for out, row in zip(called, y):
            out.append(row)

    # the same by replay
    cache = new_cache()
    replayed = [list(t.unbind()) for t in prompt(cache)]
    sx, sr = (torch.zeros((batch, hidden), dtype=torch.bfloat16, device=dev) for _ in range(2))
    slots, pos, lens = torch.full((batch,), -1, device=dev), torch.zeros(batch, dtype=torch.int64, device=dev), torch.ones(batch, dtype=torch.int32, device=dev)
    layer(sx, sr, cache, slots, pos, table, lens)  # loads the kernels; slots of -1 leave the cache alone
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y, _ = layer(sx, sr, cache, slots, pos, table, lens)
    for i in range(new_tokens):
        pos.copy_(torch.tensor([n + i for n in prompts]))
        slots.copy_(slots_of(seq, pos))
        lens.copy_(pos + 1)
        for j, n in enumerate(prompts):
            sx[j], sr[j] = x[j][n + i], res[j][n + i]
        graph.replay()
        for out, row in zip(replayed, y.clone()):
            out.append(row)

    torch.cuda.synchronize()
    start = time.perf_counter()
    for _ in range(100):  # the last token again
        graph.replay()
    torch.cuda.synchronize()
    step = (time.perf_counter() - start) / 100
    plain = layer.plain(torch.cat(x), torch.cat(res), total).split(total)
    return [torch.stack(t) for t in called], [torch.stack(t) for t in replayed], list(plain), step


def distance(outputs, plain):
    """Relative root mean square error."""
    a, b = torch.cat(outputs).float(), torch.cat(plain)
    return ((a - b).square().mean() / b.square().mean()).sqrt().item()


if __name__ == "__main__":
    args = argparse.ArgumentParser()
    for name, value in (("hidden", 4096), ("q-heads", 32), ("kv-heads", 8), ("head-dim", 128), ("tokens", 8)):
        args.add_argument("--" + name, type=int, default=value)
    args.add_argument("--prompts", type=int, nargs="+", default=[1000, 300, 64, 1])
    a = args.parse_args()
    called, replayed, plain, step = run(a.prompts, a.tokens, a.hidden, a.q_heads, a.kv_heads, a.head_dim)
    print(f"distance from float32: {distance(called, plain):.3f} by calls, {distance(replayed, plain):.3f} by replay; "
          f"{1e6 * step:.1f} us a replayed step of {len(a.prompts)} sequences")
