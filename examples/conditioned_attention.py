"""A conditioned attention block for a batch of requests, on the quantised
projections and the operators that run beside them.

Every request has its own adapter and its own text length:

* queries, keys and values are INT8 (W8A8) projections that all requests
  share, each with the request's low-rank adapter added (``lora_batched``);
* the heads of queries and keys are normalised and the queries turned by
  their positions (``qk_norm_rope``);
* the image tokens attend to their own text (``cross_attention``), and the
  output projection adds the result to the input.

``python examples/conditioned_attention.py`` runs it on random weights and
compares it with the same block in 64-bit torch arithmetic (the quantised
weights and activations taken as the values they stand for).
"""

from __future__ import annotations

import importlib
import os
import sys
import types

import torch

_ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
_PACKAGE = "comfyui-int-crush_b200"


def runtime():
    """The package's runtime (its directory name is not an identifier)."""
    if _PACKAGE not in sys.modules:
        pkg = types.ModuleType(_PACKAGE)
        pkg.__path__ = [os.path.join(_ROOT, _PACKAGE)]
        sys.modules[_PACKAGE] = pkg
    return importlib.import_module(_PACKAGE + "._b200_runtime")


class Projection:
    """An INT8 linear with per-channel scales, shared by all requests, and an
    adapter for each request beside it."""

    def __init__(self, rt, n_in, n_out, adapters, rank, gen):
        self.rt = rt
        w = torch.randn(n_out, n_in, device="cuda", generator=gen) * n_in ** -0.5
        self.w, self.s_w = rt.quantize_weight(w, 8)
        half = lambda *s, std: (torch.randn(*s, device="cuda", generator=gen) * std).half()  # noqa: E731
        self.down = half(adapters, rank, n_in, std=n_in ** -0.5)
        self.up = half(adapters, n_out, rank, std=0.3 * rank ** -0.5)
        self.scales = torch.rand(adapters, device="cuda", generator=gen) + 0.5

    def __call__(self, x, ids):
        xq, s_a = self.rt.dynamic_quantize_activation(x)
        y = self.rt.gemm_a8(xq.view(-1, x.shape[-1]), self.w, self.s_w, s_a.view(-1), out_dtype=torch.float16)
        y = y.view(*x.shape[:-1], -1)
        return self.rt.lora_batched(x, self.down, self.up, ids, self.scales, base=y, out=y)

    def plain(self, x, ids):
        xq, s_a = self.rt.dynamic_quantize_activation(x)
        y = (xq.double() @ self.w.double().T) * self.s_w.double() * s_a.double()[..., None]
        out = y.clone()
        for b, a in enumerate(ids.tolist()):
            if a >= 0:
                out[b] += self.scales[a].double() * ((x[b].double() @ self.down[a].double().T) @ self.up[a].double().T)
        return out


class ConditionedAttention:
    def __init__(self, hidden=1024, heads=16, key_heads=4, text=768, adapters=3, rank=16, positions=4096, seed=0):
        self.rt = rt = runtime()
        gen = torch.Generator(device="cuda").manual_seed(seed)
        self.heads, self.key_heads, self.d = heads, key_heads, hidden // heads
        self.q = Projection(rt, hidden, hidden, adapters, rank, gen)
        self.kv = Projection(rt, text, 2 * key_heads * self.d, adapters, rank, gen)
        self.o = Projection(rt, hidden, hidden, adapters, rank, gen)
        self.q_gamma = 1 + 0.1 * torch.randn(self.d, device="cuda", generator=gen)
        self.k_gamma = 1 + 0.1 * torch.randn(self.d, device="cuda", generator=gen)
        freq = 10000.0 ** (-torch.arange(0, self.d, 2, device="cuda", dtype=torch.float64) / self.d)
        angle = torch.arange(positions, device="cuda", dtype=torch.float64)[:, None] * freq
        self.cos, self.sin = angle.cos().float(), angle.sin().float()

    def __call__(self, x, text, text_lens, ids, positions=None):
        """x [B, L, hidden] and text [B, T, text] in fp16, text_lens [B], an
        adapter id per request (-1: none) -> [B, L, hidden]."""
        B, L, _ = x.shape
        q = self.q(x, ids).view(B, L, self.heads, self.d)
        kv = self.kv(text, ids).view(B, -1, 2, self.key_heads, self.d)
        q = self.rt.qk_norm_rope(q, q_gamma=self.q_gamma, cos=self.cos, sin=self.sin, positions=positions)
        k = self.rt.qk_norm_rope(kv[:, :, 0], q_gamma=self.k_gamma)
        a = self.rt.cross_attention(q, k, kv[:, :, 1], kv_lens=text_lens)
        return x + self.o(a.view(B, L, -1), ids)

    def plain(self, x, text, text_lens, ids):
        """The same in 64 bits, rounded where the block hands fp16 on."""
        B, L, _ = x.shape
        norm = lambda t, g: t / torch.sqrt((t * t).mean(-1, keepdim=True) + 1e-6) * g.double()  # noqa: E731
        q = norm(self.q.plain(x, ids).half().double().view(B, L, self.heads, self.d), self.q_gamma)
        c, s = self.cos[:L].double()[:, None], self.sin[:L].double()[:, None]
        q = torch.stack([q[..., 0::2] * c - q[..., 1::2] * s, q[..., 1::2] * c + q[..., 0::2] * s], -1).flatten(-2)
        kv = self.kv.plain(text, ids).half().double().view(B, -1, 2, self.key_heads, self.d)
        k, v = norm(kv[:, :, 0], self.k_gamma), kv[:, :, 1]
        group = self.heads // self.key_heads
        k, v = (t.repeat_interleave(group, 2).transpose(1, 2) for t in (k, v))
        scores = q.transpose(1, 2) @ k.transpose(2, 3) * self.d ** -0.5
        hidden = torch.arange(text.shape[1], device=x.device) >= text_lens.view(-1, 1, 1, 1)
        p = torch.softmax(scores.masked_fill(hidden, -torch.inf), -1).nan_to_num(0.0)
        a = (p @ v).transpose(1, 2).reshape(B, L, -1).half()
        return x.double() + self.o.plain(a, ids)


def main():
    block = ConditionedAttention()
    gen = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randn(4, 500, 1024, device="cuda", generator=gen).half()
    text = torch.randn(4, 77, 768, device="cuda", generator=gen).half()
    lens = torch.tensor([77, 12, 0, 30], device="cuda")   # one request without text
    ids = torch.tensor([2, 0, 1, -1], device="cuda")      # one without an adapter
    out = block(x, text, lens, ids)
    want = block.plain(x, text, lens, ids)
    error = ((out.double() - want).norm() / want.norm()).item()
    print(f"conditioned attention block: relative error {error:.2e}")
    return error


if __name__ == "__main__":
    main()
