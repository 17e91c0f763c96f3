"""A decoder layer of the architecture put together from this library's operators: several requests, each with an adapter of its own or none.

    python examples/decoder_layer.py [--requests 8] [--prompt 300] [--steps 16] [--bits4]

  x -> RMSNorm -> QKV projection + adapters -> cache append and attention -> O projection + adapters -> + x
    -> RMSNorm -> router -> routed experts (and one shared expert) -> + x
  rows -> RMSNorm -> output head -> log probabilities of a token, entropy, the best alternatives

The norms and residuals are torch's; everything that picks its weights row by row, the attention, and what is asked of the logits is `hy3_b200`.  The shared
projections are torch's on bf16 weights, with --bits4 `hy3_b200.linear4`'s on weights in 4 bits, as the output head's always are.
Weights are random.  A prompt goes through in one chunk per request, then all requests go on token by token together.
"""
import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
import hy3_b200  # noqa: E402
from hy3_b200 import D, G, H, Hy3Attn  # noqa: E402


def rms_norm(x, weight, eps=1e-5):
    return x * torch.rsqrt(x.square().mean(-1, keepdim=True) + eps) * weight


class DecoderLayer:
    """One layer.  Activations are bf16 between the operators and fp32 in the residual stream; rows are [n, hidden] fp32."""

    def __init__(self, hidden=4096, experts=192, top_k=8, inter=1536, adapters=4, rank=16, requests=8, max_tokens_per_seq=4096, chunk=512, kv_dtype="int8", seed=0, device="cuda", bits4=False):
        gen = torch.Generator(device=device).manual_seed(seed)

        def weight(*shape, scale=None):
            w = torch.randn(shape, device=device, dtype=torch.bfloat16, generator=gen)
            return w.mul_(shape[-1] ** -0.5 if scale is None else scale)
        self.hidden, self.top_k, self.chunk = hidden, top_k, chunk
        self.norm1, self.norm2 = 1 + 0.02 * weight(hidden, scale=1).float(), 1 + 0.02 * weight(hidden, scale=1).float()
        self.qkv, self.o = weight((H + 2 * G) * D, hidden), weight(hidden, H * D)
        self.qkv_a, self.qkv_b = weight(adapters, rank, hidden), weight(adapters, (H + 2 * G) * D, rank)
        self.o_a, self.o_b = weight(adapters, rank, H * D), weight(adapters, hidden, rank)
        self.scales = 0.25 + 0.5 * torch.rand(adapters, device=device, generator=gen)
        self.router, self.bias = weight(experts, hidden).float(), 0.05 * torch.randn(experts, device=device, generator=gen)
        self.gate, self.up, self.down = weight(experts, inter, hidden), weight(experts, inter, hidden), weight(experts, hidden, inter)
        self.shared_gate, self.shared_up, self.shared_down = weight(inter, hidden), weight(inter, hidden), weight(hidden, inter)
        shared = {"qkv": self.qkv, "o": self.o, "gate": self.shared_gate, "up": self.shared_up, "down": self.shared_down}
        self.bits4 = {name: hy3_b200.quantize4(w) for name, w in shared.items()} if bits4 else None
        if bits4:           # (what they were made of is not kept)
            self.qkv = self.o = self.shared_gate = self.shared_up = self.shared_down = None
        self.ctx = Hy3Attn(kv_dtype=kv_dtype, n_layers=1, max_seqs=requests, max_batch=max(chunk, requests), max_tokens=requests * max_tokens_per_seq,
                           max_tokens_per_seq=max_tokens_per_seq)
        self.q16 = torch.empty((chunk, H, D), dtype=torch.float16, device=device)

    def close(self):
        self.ctx.close()

    def shared(self, name, weight, x, out_dtype=torch.bfloat16):
        """Rows x times a weight that all rows share."""
        return torch.mm(x, weight.T).to(out_dtype) if self.bits4 is None else hy3_b200.linear4(x, *self.bits4[name], out_dtype=out_dtype)

    def project(self, x, adapter):
        """q [n, 64, 128], k and v [n, 8, 128] of rows x, views of one projection's rows (as the attention takes them)."""
        h = rms_norm(x, self.norm1).bfloat16()
        rows = self.shared("qkv", self.qkv, h, torch.float32)
        hy3_b200.adapters(h, rows, self.qkv_a, self.qkv_b, adapter, self.scales, out=rows)
        q, k, v = rows.split([H * D, G * D, G * D], dim=1)
        return q.unflatten(1, (H, D)), k.unflatten(1, (G, D)), v.unflatten(1, (G, D))

    def finish(self, x, attn, adapter):
        """The layer behind the attention; returns the rows, and the experts and weights they went through."""
        a = attn.flatten(1).bfloat16()
        x = x + hy3_b200.adapters(a, self.shared("o", self.o, a), self.o_a, self.o_b, adapter, self.scales).float()
        h = rms_norm(x, self.norm2)
        ids, weights = hy3_b200.route(h @ self.router.T, self.bias, top_k=self.top_k, score="sigmoid", scale=2.826)
        h = h.bfloat16()
        routed = hy3_b200.experts(h, ids, weights, self.gate, self.up, self.down)
        gated = torch.nn.functional.silu(self.shared("gate", self.shared_gate, h)) * self.shared("up", self.shared_up, h)
        shared = self.shared("down", self.shared_down, gated)
        return x + routed.float() + shared.float(), ids, weights

    def prompt(self, seq, x, adapter, routed=None):
        """Rows x of a fresh request `seq`, with its adapter (-1: none), in chunks; each chunk's experts and weights are appended to `routed`."""
        out = []
        for t in range(0, x.shape[0], self.chunk):
            part = x[t:t + self.chunk]
            n = part.shape[0]
            which = torch.full((n,), adapter, dtype=torch.int32, device=x.device)
            self.ctx.batch_set([seq] * n, list(range(t, t + n)))
            q, k, v = self.project(part, which)
            self.ctx.append(0, q, k, v, q_out=False, q_out16=self.q16[:n])
            rows, *experts = self.finish(part, self.ctx.prefill(0, seq, t, self.q16[:n]), which)
            out.append(rows)
            if routed is not None:
                routed.append(experts)
        return torch.cat(out)

    def step(self, seqs, slots, x, adapter):
        """One new row x[i] of each request seqs[i] at position slots[i], adapter int32 [n]."""
        self.ctx.batch_set(seqs, slots)
        return self.finish(x, self.ctx.decode_step(0, *self.project(x, adapter)), adapter)


class OutputHead:
    """The model's last norm and its output head in 4 bits."""

    def __init__(self, hidden=4096, vocab=120832, group=64, seed=1, device="cuda"):
        gen = torch.Generator(device=device).manual_seed(seed)
        self.norm = 1 + 0.02 * torch.randn(hidden, device=device, generator=gen)
        self.codes, self.scales = hy3_b200.quantize4(torch.randn((vocab, hidden), device=device, dtype=torch.bfloat16, generator=gen).mul_(2.5 * hidden ** -0.5), group=group)

    def logits(self, x):
        """fp32 logits [n, vocab] of rows x [n, hidden]."""
        return hy3_b200.linear4(rms_norm(x, self.norm).bfloat16(), self.codes, self.scales, out_dtype=torch.float32)

    def answer(self, x, tokens=None, top_k=5):
        """Of rows x: log probabilities of the tokens, entropies, the best alternatives and their log probabilities."""
        return hy3_b200.logprobs(self.logits(x), tokens, top_k)


def main():
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--requests", type=int, default=8)
    ap.add_argument("--prompt", type=int, default=300)
    ap.add_argument("--steps", type=int, default=16)
    ap.add_argument("--bits4", action="store_true", help="shared projections on weights in 4 bits")
    a = ap.parse_args()
    layer, head = DecoderLayer(requests=a.requests, max_tokens_per_seq=a.prompt + a.steps + 128, bits4=a.bits4), OutputHead()
    adapter = torch.arange(a.requests, device="cuda", dtype=torch.int32) % 5 - 1
    for s in range(a.requests):
        layer.prompt(s, torch.randn((a.prompt, layer.hidden), device="cuda"), s % 5 - 1)
    begin, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    for i in range(a.steps):
        if i == a.steps // 2:
            begin.record()
        rows, ids, _ = layer.step(list(range(a.requests)), [a.prompt + i] * a.requests, torch.randn((a.requests, layer.hidden), device="cuda"), adapter)
        _, entropy, best, logp = head.answer(rows)
    end.record()
    layer.ctx.sync()
    hy3_b200.layer_sync()
    print("%d requests behind %d tokens: %.0f us a step; first row through experts %s, norm %.3f" % (
        a.requests, a.prompt, begin.elapsed_time(end) * 1000 / (a.steps - a.steps // 2), ids[0].tolist(), float(rows[0].norm())))
    print("its best tokens %s, log probabilities %s, entropy %.2f" % (best[0].tolist(), ["%.2f" % v for v in logp[0].tolist()], float(entropy[0])))
    layer.close()


if __name__ == "__main__":
    main()
