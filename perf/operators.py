"""Workloads of the attention-side operators: what runs beside the quantised
projections of a conditioned transformer block.

* ``qk``: RMS norm of every query and key head and the position rotation, in
  one pass over the projection's output;
* ``attn``: cross attention of image / decoder tokens to an encoder's states
  of another length, with per-sample lengths or key masks;
* ``lora``: the low-rank adapters of many requests at once, added beside a
  shared projection.

``own`` false computes them as elementary torch operations in 32 bits,
``own`` true as calls of the package's entry points.
"""

import importlib
import math
import os
import sys
import types

import torch

own = False

_DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}
_ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
_PACKAGE = "comfyui-int-crush_b200"


def _runtime():
    """The package's runtime (its directory name is not an identifier)."""
    if _PACKAGE not in sys.modules:
        pkg = types.ModuleType(_PACKAGE)
        pkg.__path__ = [os.path.join(_ROOT, _PACKAGE)]
        sys.modules[_PACKAGE] = pkg
    return importlib.import_module(_PACKAGE + "._b200_runtime")


# ── cases ────────────────────────────────────────────────────────────────────

def _qk(name, B, L, H, Hk, D, rot, layout, dtype, positions):
    return {"name": name, "op": "qk", "B": B, "L": L, "H": H, "Hk": Hk, "D": D, "rot": rot, "layout": layout,
            "dtype": dtype, "positions": positions}


def _attn(name, B, Lq, Lk, H, Hk, D, dtype, mask):
    return {"name": name, "op": "attn", "B": B, "Lq": Lq, "Lk": Lk, "H": H, "Hk": Hk, "D": D, "dtype": dtype,
            "mask": mask}


def _lora(name, S, rows, K, N, R, n, dtype, packed):
    return {"name": name, "op": "lora", "S": S, "rows": rows, "K": K, "N": N, "R": R, "n": n, "dtype": dtype,
            "packed": packed}


def listed():
    return [
        # one new token of a batch of four, queries sharing key heads: the
        # smallest call, where the launch is what it costs
        _qk("qk_token", 4, 1, 32, 8, 128, 128, "half", "bf16", True),
        # a ragged batch with only half of each head rotated, at positions
        # that do not start at zero
        _qk("qk_partial_ragged", 3, 1001, 32, 8, 96, 48, "half", "fp16", True),
        # the joint sequence of a double-stream image block: 4096 image and
        # 512 text tokens, 24 heads of 128
        _qk("qk_image_block", 1, 4608, 24, 24, 128, 128, "interleaved", "fp16", False),
        # a video block: 32760 tokens, 40 heads of 128, batch 2
        _qk("qk_video_block", 2, 32760, 40, 40, 128, 128, "interleaved", "bf16", False),
        # one query token against a short text: latency
        _attn("attn_token_short", 1, 1, 77, 8, 8, 64, "fp16", "none"),
        # single decoder tokens of eight requests, each over its own encoder
        # length up to 8192, grouped key heads: the cache's bytes count
        _attn("attn_token_long", 8, 1, 8192, 32, 8, 128, "bf16", "lens"),
        # odd lengths, one sample without any key, keys dropped one by one
        _attn("attn_odd_masked", 3, 1023, 333, 20, 20, 64, "fp16", "bool"),
        # an image block's tokens over 512 text states with an additive mask
        # whose padding holds the type's lowest value
        _attn("attn_image_text", 2, 4096, 512, 24, 24, 128, "bf16", "add"),
        # a video block's 32760 tokens over 512 text states, 40 heads, batch 2
        _attn("attn_video_text", 2, 32760, 512, 40, 40, 128, "bf16", "none"),
        # sixteen requests of one token, eight adapters: adapter bytes count
        _lora("lora_tokens", 16, 1, 5120, 5120, 16, 8, "bf16", False),
        # ragged requests packed into one batch, a rank that is no power of two
        _lora("lora_ragged_packed", 2777, 1, 5120, 5120, 24, 4, "fp16", True),
        # eight video samples, an adapter each, before the wide FFN projection
        _lora("lora_video_ffn", 8, 4095, 5120, 13824, 32, 6, "bf16", False),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.99))))))


def draw(rng):
    dtype = rng.choice(["fp16", "bf16"])
    op = rng.choice(["qk", "attn", "lora"])
    if op == "qk":
        Hk = rng.choice([1, 2, 3, 5, 8, 10, 20])
        H = Hk * rng.choice([1, 1, 2, 4])
        D = rng.choice([40, 64, 72, 80, 96, 128, 128, 256])
        rot = rng.choice([D, D, D // 2 // 2 * 2, 16])
        B = _log(rng, 1, 8)
        most = 2 * 32760 * 80 * 128 // (B * (H + Hk) * D)
        c = _qk("", B, _log(rng, 1, min(32760, most)), H, Hk, D, rot, rng.choice(["half", "interleaved"]), dtype,
                rng.random() < 0.5)
    elif op == "attn":
        Hk = rng.choice([1, 2, 3, 5, 8, 10, 20])
        H = Hk * rng.choice([1, 1, 2, 4])
        D = rng.choice([40, 64, 80, 96, 128, 128])
        B = _log(rng, 1, 8)
        Lk = _log(rng, 1, 16384)
        most = 2 * 32760 * 512 * 40 * 128 // (B * Lk * H * D)
        Lq = 1 if rng.random() < 0.25 else _log(rng, 1, max(1, min(32760, most)))
        c = _attn("", B, Lq, Lk, H, Hk, D, dtype, rng.choice(["none", "lens", "bool", "add"]))
    else:
        K, N = (_log(rng, 64, 1728) * 8 - rng.choice([0, 0, 0, 0, 3]) for _ in range(2))
        R = rng.choice([4, 8, 12, 16, 24, 32, 64, 128])
        n = _log(rng, 1, 16)
        most = 8 * 4095 * (5120 + 2 * 13824) // (K + 2 * N)
        if rng.random() < 0.3:
            c = _lora("", _log(rng, 65, min(most, 6000)), 1, K, N, R, min(n, 8), dtype, True)
        else:
            rows = 1 if rng.random() < 0.4 else _log(rng, 1, 4096)
            c = _lora("", _log(rng, 1, max(1, min(64, most // rows))), rows, K, N, R, n, dtype, False)
    del c["name"]
    return c


# ── inputs ───────────────────────────────────────────────────────────────────

def _lengths(c):
    """Keys that each sample of an attention case sees (before shuffling):
    spread down from all of them; the last sample of a masked batch of three
    or more sees none."""
    B, Lk = c["B"], c["Lk"]
    if c["mask"] == "none":
        return [Lk] * B
    got = [max(1, Lk - b * Lk // B) for b in range(B)]
    if c["mask"] == "bool" and B >= 3:
        got[-1] = 0
    return got


def _bare(c):
    """Requests of a lora case that have no adapter: every eighth."""
    return c["S"] // 8


def prepare(case, seed):
    c = case
    dev = "cuda"
    dt = _DTYPES[c["dtype"]]
    g = torch.Generator(device=dev)
    g.manual_seed(seed)

    def normal(*shape, std=1.0, mean=0.0):
        t = torch.empty(shape, dtype=dt, device=dev)
        return t.normal_(mean, std, generator=g)

    if c["op"] == "qk":
        # the fused projection's output, queries, keys and values side by side
        B, L, H, Hk, D = c["B"], c["L"], c["H"], c["Hk"], c["D"]
        qkv = normal(B, L, (H + 2 * Hk) * D, std=1.5)
        s = {"q": qkv[..., :H * D].view(B, L, H, D), "k": qkv[..., H * D:(H + Hk) * D].view(B, L, Hk, D)}
        s["q_gamma"] = torch.empty(D, device=dev).normal_(1.0, 0.2, generator=g)
        s["k_gamma"] = torch.empty(D, device=dev).normal_(1.0, 0.2, generator=g)
        table = L + 4096 if c["positions"] else L
        inv = 10000.0 ** (-torch.arange(0, c["rot"], 2, device=dev, dtype=torch.float64) / c["rot"])
        a = torch.arange(table, device=dev, dtype=torch.float64)[:, None] * inv
        s["cos"], s["sin"] = a.cos().float(), a.sin().float()
        s["positions"] = None
        if c["positions"]:
            start = torch.randint(0, 4097, (B, 1), device=dev, generator=g)
            s["positions"] = (start + torch.arange(L, device=dev)).to(torch.int32)
        s["layout"] = c["layout"]
    elif c["op"] == "attn":
        B, Lq, Lk, H, Hk, D = c["B"], c["Lq"], c["Lk"], c["H"], c["Hk"], c["D"]
        s = {"q": normal(B, Lq, H, D)}
        # keys and values of one fused projection of the encoder's states
        kv = normal(B, Lk, 2, Hk, D)
        kv[:, :, 1] += 0.25
        s["k"], s["v"] = kv[:, :, 0], kv[:, :, 1]
        s["kv_lens"] = s["key_mask"] = None
        order = torch.randperm(B, device=dev, generator=g)
        lens = torch.tensor(_lengths(c), device=dev)[order]
        if c["mask"] == "lens":
            s["kv_lens"] = lens.to(torch.int32)
        elif c["mask"] == "bool":
            rank = torch.rand(B, Lk, device=dev, generator=g).argsort(1).argsort(1)
            s["key_mask"] = rank < lens[:, None]
        elif c["mask"] == "add":
            seen = torch.arange(Lk, device=dev) < lens[:, None]
            s["key_mask"] = torch.where(seen, normal(B, Lk), torch.finfo(dt).min)
    else:
        S, rows, K, N, R, n = c["S"], c["rows"], c["K"], c["N"], c["R"], c["n"]
        M = S * rows
        s = {"x": normal(M, K), "base": normal(M, N)}
        s["down"] = normal(n, R, K, std=K ** -0.5)
        s["up"] = normal(n, N, R, std=0.5 * R ** -0.5)
        s["scales"] = torch.empty(n, device=dev).uniform_(0.5, 1.5, generator=g)
        ids = torch.arange(S, device=dev) % n
        ids[:_bare(c)] = -1
        if c["packed"]:
            # requests of uneven lengths: runs of rows with the same adapter
            ids = ids.sort().values.roll(int(torch.randint(0, S, (1,), generator=g, device=dev)))
        else:
            ids = ids[torch.randperm(S, device=dev, generator=g)]
        s["ids"] = ids.to(torch.int32)
        s["packed"] = c["packed"]
    s["op"] = c["op"]
    return s


# ── one pass ─────────────────────────────────────────────────────────────────

def _plain_norm_rotate(x, gamma, cos, sin, layout):
    x = x.float()
    x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-6) * gamma
    rot = 2 * cos.shape[-1]
    t, rest = x[..., :rot], x[..., rot:]
    if layout == "half":
        a, b = t[..., :rot // 2], t[..., rot // 2:]
        t = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    else:
        a, b = t[..., 0::2], t[..., 1::2]
        t = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    return torch.cat([t, rest], -1)


def _plain_attention(q, k, v, kv_lens, key_mask):
    B, Lq, H, D = q.shape
    Lk, Hk = k.shape[1:3]
    qf = q.float().permute(0, 2, 1, 3).reshape(B, Hk, H // Hk * Lq, D)
    kf, vf = k.float().permute(0, 2, 1, 3), v.float().permute(0, 2, 1, 3)
    s = (qf * D ** -0.5) @ kf.transpose(-1, -2)
    if kv_lens is not None:
        s = s.masked_fill(torch.arange(Lk, device=q.device) >= kv_lens.view(B, 1, 1, 1), -math.inf)
    if key_mask is not None and key_mask.dtype == torch.bool:
        s = s.masked_fill(~key_mask.view(B, 1, 1, Lk), -math.inf)
    elif key_mask is not None:
        s = s + key_mask.float().view(B, 1, 1, Lk)
    m = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(m == -math.inf, 0.0, m))
    total = p.sum(-1, keepdim=True)
    o = (p @ vf) / torch.where(total == 0, 1.0, total)
    return o.view(B, H, Lq, D).transpose(1, 2).contiguous().to(q.dtype)


def _plain_lora(x, base, down, up, ids, scales, packed):
    M, S, R = x.shape[0], ids.shape[0], down.shape[1]
    factor = torch.where(ids < 0, 0.0, scales[ids.clamp(min=0).long()])
    pick = ids.clamp(min=0).long()
    if packed:
        # every adapter on every row, the others' parts set to zero
        one = torch.nn.functional.one_hot(pick, down.shape[0]) * factor[:, None]
        mid = (x.float() @ down.float().flatten(0, 1).T).view(M, -1, R) * one[..., None]
        y = mid.flatten(1) @ up.float().transpose(1, 2).flatten(0, 1)
    else:
        mid = x.float().view(S, M // S, -1) @ down.float()[pick].transpose(1, 2) * factor.view(S, 1, 1)
        y = (mid @ up.float()[pick].transpose(1, 2)).view(M, -1)
    return (base.float() + y).to(x.dtype)


def run(state):
    s = state
    if own:
        rt = _runtime()
        if s["op"] == "qk":
            return rt.qk_norm_rope(s["q"], s["k"], q_gamma=s["q_gamma"], k_gamma=s["k_gamma"], cos=s["cos"],
                                   sin=s["sin"], layout=s["layout"], positions=s["positions"], eps=1e-6)
        if s["op"] == "attn":
            return rt.cross_attention(s["q"], s["k"], s["v"], kv_lens=s["kv_lens"], key_mask=s["key_mask"])
        return rt.lora_batched(s["x"], s["down"], s["up"], s["ids"], s["scales"], base=s["base"])
    if s["op"] == "qk":
        cos, sin = s["cos"], s["sin"]
        if s["positions"] is not None:
            cos, sin = cos[s["positions"]], sin[s["positions"]]
        cos, sin = cos.unsqueeze(-2), sin.unsqueeze(-2)
        return tuple(_plain_norm_rotate(s[t], s[t + "_gamma"], cos, sin, s["layout"]).to(s[t].dtype) for t in "qk")
    if s["op"] == "attn":
        return _plain_attention(s["q"], s["k"], s["v"], s["kv_lens"], s["key_mask"])
    return _plain_lora(s["x"], s["base"], s["down"], s["up"], s["ids"], s["scales"], s["packed"])


# ── what a pass cannot do without ────────────────────────────────────────────

def work(case):
    c = case
    if c["op"] == "qk":
        rows = c["B"] * c["L"] * (c["H"] + c["Hk"])
        # rows in and out, the table rows that the positions name, positions
        table = c["L"] if not c["positions"] else min(c["B"] * c["L"], c["L"] + 4096)
        other = 2 * c["D"] * 4 + table * c["rot"] * 4 + (c["B"] * c["L"] * 4 if c["positions"] else 0)
        return {"bytes": rows * c["D"] * 4 + other, "flops": rows * (4 * c["D"] + 3 * c["rot"])}
    if c["op"] == "attn":
        seen = sum(_lengths(c))
        mask = {"none": 0, "lens": 4 * c["B"], "bool": c["B"] * c["Lk"], "add": 2 * c["B"] * c["Lk"]}[c["mask"]]
        return {"bytes": 4 * c["B"] * c["Lq"] * c["H"] * c["D"] + 4 * seen * c["Hk"] * c["D"] + mask,
                "flops": 4 * seen * c["Lq"] * c["H"] * c["D"]}
    M, used = c["S"] * c["rows"], min(c["n"], c["S"] - _bare(c))
    active = (c["S"] - _bare(c)) * c["rows"]
    return {"bytes": 2 * active * c["K"] + 4 * M * c["N"] + 2 * used * c["R"] * (c["K"] + c["N"]) + 4 * c["S"],
            "flops": 2 * active * c["R"] * (c["K"] + c["N"])}


# ── the definitions in 64 bits ───────────────────────────────────────────────

def exact(case, seed):
    s = prepare(case, seed)
    f = torch.float64
    if case["op"] == "qk":
        got = []
        for t in "qk":
            # as complex numbers: the pair (a, b) turns by the position's angle
            x = s[t].to(f)
            x = x / (x.square().sum(-1, keepdim=True) / x.shape[-1] + 1e-6).sqrt() * s[t + "_gamma"].to(f)
            turn = torch.complex(s["cos"].to(f), s["sin"].to(f))
            at = torch.arange(x.shape[1], device=x.device) if s["positions"] is None else s["positions"].long()
            turn = turn[at][..., None, :]
            h = case["rot"] // 2
            i = torch.arange(h, device=x.device)
            first, second = (i, i + h) if case["layout"] == "half" else (2 * i, 2 * i + 1)
            z = torch.complex(x[..., first], x[..., second]) * turn
            x[..., first], x[..., second] = z.real, z.imag
            got.append(x)
        return tuple(got)
    if case["op"] == "attn":
        B, Lq, H, D = s["q"].shape
        group = H // case["Hk"]
        out = torch.zeros(B, Lq, H, D, dtype=f, device="cuda")
        for b in range(B):
            add = torch.zeros(case["Lk"], dtype=f, device="cuda")
            keep = torch.ones(case["Lk"], dtype=torch.bool, device="cuda")
            if s["kv_lens"] is not None:
                keep[int(s["kv_lens"][b]):] = False
            if case["mask"] == "bool":
                keep = s["key_mask"][b]
            elif case["mask"] == "add":
                add = s["key_mask"][b].to(f)
            if not bool(keep.any()):
                continue
            for h in range(H):
                k, v = s["k"][b, keep, h // group].to(f), s["v"][b, keep, h // group].to(f)
                w = torch.softmax(torch.addmm(add[keep], s["q"][b, :, h].to(f), k.T, alpha=1 / math.sqrt(D)), -1)
                out[b, :, h] = w @ v
        return out
    x, out = s["x"].to(f), s["base"].to(f)
    of_row = s["ids"].long().repeat_interleave(case["rows"])
    for i in range(case["n"]):
        rows = (of_row == i).nonzero()[:, 0]
        out[rows] += s["scales"][i].to(f) * ((x[rows] @ s["down"][i].to(f).T) @ s["up"][i].to(f).T)
    return out
