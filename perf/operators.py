"""Timing cases of the prompt, draft and cache operators.

* ``prompt``  causal attention over whole prompts (``turboquant.runtime.prompt_attention``): one prompt,
              a padded batch, and prompts of different lengths packed behind one another;
* ``tree``    attention of a tree of drafted tokens over a packed cache
              (``turboquant.runtime.kernels.tree_attention``);
* ``keep``    the accepted path of a drafted tree moved together in its cache, in place
              (``turboquant.runtime.kernels.keep_tokens``);
* ``gather``  a new cache of chosen batch rows and tokens (``turboquant.runtime.kernels.gather_tokens``).

Head dimension 128 throughout.  Queries are N(0, 1); keys and values have iid N(0, 1) directions, packed
ones with lognormal norms around 20.  Packed caches are quantized here with elementary operations: a
random rotation, Lloyd-Max codes of a coordinate, fp16 norms and, with QJL, the signs of a Gaussian
sketch of the key's residual and its fp16 norm.
"""

from __future__ import annotations

import functools
import math
import sys
from pathlib import Path

import numpy as np
import torch

#: where this repository keeps its package
_PACKAGE = str(Path(__file__).resolve().parent.parent / "tq-local_amd")
if _PACKAGE not in sys.path:
    sys.path.insert(0, _PACKAGE)

own = False

D = 128
DEV = "cuda"


# ---------------------------------------------------------------- cases


def _prompt(name, lens, Hq, Hkv, dtype="bf16", packed=False, tail=0):
    """``lens`` as text, e.g. "301" or "1500 1211"; packed: behind one another, with ``tail`` unused rows."""
    c = {"op": "prompt", "lens": lens, "Hq": Hq, "Hkv": Hkv, "dtype": dtype, "packed": packed, "tail": tail}
    return dict(c, name=name) if name else c


def _tree(name, B, Hq, Hkv, N, T, shape, bits, qjl, ragged=False):
    c = {"op": "tree", "B": B, "Hq": Hq, "Hkv": Hkv, "N": N, "T": T, "shape": shape, "bits": bits, "qjl": qjl,
         "ragged": ragged}
    return dict(c, name=name) if name else c


def _moves(name, op, B, Hkv, N, bits, qjl, split=0, rows=0, keep=0, T=0):
    c = {"op": op, "B": B, "Hkv": Hkv, "N": N, "bits": bits, "qjl": qjl, "split": split, "rows": rows, "keep": keep,
         "T": T}
    return dict(c, name=name) if name else c


def listed():
    return [
        # one short prompt of odd length, 32 query heads on 8 KV heads: the smallest, latency counts
        _prompt("prompt_short", "301", 32, 8),
        # one prompt of 8K tokens
        _prompt("prompt_8k", "8192", 32, 8),
        # the longest prompt
        _prompt("prompt_16k", "16384", 32, 8),
        # prompts of a serving queue packed behind one another, one of them empty and one of one token;
        # 7 query heads per KV head
        _prompt("prompt_packed", "2811 0 517 1 1403 96 733 450", 28, 4, packed=True, tail=37),
        # a left-padded batch of a fp16 model, 5 query heads per KV head
        _prompt("prompt_padded_fp16", "1500 1211 640 27", 40, 8, dtype="fp16"),
        # 8 drafted tokens of one short chat, 4-bit Q_prod: the smallest
        _tree("tree_short_chat", 1, 32, 8, 1037, 8, "tree", 4, True),
        # 16 drafted tokens for each of 8 sequences at 32K: the largest cache
        _tree("tree_8b_32k", 8, 32, 8, 32768, 16, "tree", 4, True),
        # a wide tree, 3-bit Q_mse, 7 query heads per KV head
        _tree("tree_wide_3bit", 4, 28, 4, 8192, 64, "tree", 3, False),
        # 5 tokens in a chain, each sequence with a range of its own; 5 query heads per KV head
        _tree("tree_chain_ragged", 3, 40, 8, 20011, 5, "chain", 4, True, ragged=True),
        # the accepted path of 16 drafted tokens behind an 8K history: latency counts
        _moves("keep_path", "keep", 1, 8, 8192, 4, True, keep=6, T=16),
        # 8 beams from 4 prompts of 32K
        _moves("gather_beams", "gather", 4, 8, 32768, 4, True, rows=8),
        # half of the history chosen for each head, a layer in two channel groups (rows of odd sizes)
        _moves("gather_half_split", "gather", 2, 8, 16384, 4, True, split=4, keep=8192),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("prompt", "prompt", "prompt", "tree", "tree", "tree", "keep", "gather"))
    Hkv, g = rng.choice(((8, 4), (4, 7), (8, 5), (2, 8), (4, 1), (8, 2)))
    qjl = rng.random() < 0.6
    bits = rng.choice((3, 4, 4)) if qjl else rng.choice((2, 3, 4))
    if op == "prompt":
        dtype = rng.choice(("bf16", "bf16", "fp16"))
        kind = rng.choice(("one", "padded", "packed"))
        if kind == "one":
            return _prompt(None, str(_log(rng, 16, 12000)), Hkv * g, Hkv, dtype)
        lens = [_log(rng, 1, 2000) for _ in range(rng.randint(2, 6))]
        if kind == "packed" and rng.random() < 0.3:
            lens[rng.randrange(len(lens))] = 0
        return _prompt(None, " ".join(map(str, lens)), Hkv * g, Hkv, dtype, kind == "packed",
                       rng.randint(0, 70) if kind == "packed" else 0)
    if op == "tree":
        return _tree(None, rng.choice((1, 2, 3, 4)), Hkv * g, Hkv, _log(rng, 64, 32768), _log(rng, 1, 64),
                     rng.choice(("tree", "chain")), bits, qjl, rng.random() < 0.4)
    if op == "keep":
        T = rng.randint(3, 64)
        return _moves(None, op, rng.choice((1, 2, 4)), Hkv, _log(rng, 64, 32768), bits, qjl,
                      keep=rng.randint(1, max(1, T // 2)), T=T)
    split = rng.choice((3, 4, 8)) if rng.random() < 0.3 else 0
    B, N = rng.choice((1, 2, 3)), _log(rng, 256, 32768)
    if rng.random() < 0.5:
        return _moves(None, op, B, Hkv, N, bits, qjl, split, rows=rng.randint(1, 6))
    return _moves(None, op, B, Hkv, N, bits, qjl, split, keep=rng.randint(1, N))


# ---------------------------------------------------------------- preparing


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _lens(c):
    return [int(x) for x in c["lens"].split()]


def _dtype(c):
    return torch.float16 if c["dtype"] == "fp16" else torch.bfloat16


def _prepare_prompt(c, seed):
    gen, lens = _gen(seed), _lens(c)
    B, S = (1, sum(lens) + c["tail"]) if c["packed"] else (len(lens), max(lens))
    s = {}
    for name, heads in (("q", c["Hq"]), ("k", c["Hkv"]), ("v", c["Hkv"])):
        # a projection's output, token by token, seen head by head
        x = torch.randn(B, S, heads, D, generator=gen, device=DEV).to(_dtype(c))
        s[name] = x.transpose(1, 2)
    if c["packed"]:
        s["cu_seqlens"] = torch.tensor(np.cumsum([0] + lens), dtype=torch.int32, device=DEV)
    elif len(lens) > 1:
        s["seq_starts"] = torch.tensor([S - n for n in lens], dtype=torch.int32, device=DEV)
    return s


@functools.lru_cache(maxsize=None)
def _codebook(bits, dim):
    """Lloyd-Max centers and their midpoints for one coordinate of a unit vector of ``dim`` coordinates."""
    x = np.linspace(-1.0, 1.0, 20001)
    p = np.maximum(1.0 - x * x, 0.0) ** ((dim - 3) / 2)
    cdf = np.cumsum(p) / p.sum()
    centers = np.interp((np.arange(1 << bits) + 0.5) / (1 << bits), cdf, x)
    for _ in range(300):
        cell = np.searchsorted((centers[1:] + centers[:-1]) / 2, x)
        mass = np.bincount(cell, p, minlength=1 << bits)
        centers = np.where(mass > 0, np.bincount(cell, p * x, minlength=1 << bits) / np.maximum(mass, 1e-300), centers)
    centers = centers.astype(np.float32)
    return centers, ((centers[1:] + centers[:-1]) / 2).astype(np.float32)


def _pack(codes, bits):
    """[..., n] codes -> the rows' LSB-first bit streams, uint8."""
    b = (codes.unsqueeze(-1) >> torch.arange(bits, device=DEV, dtype=torch.uint8)) & 1
    b = b.flatten(-2)
    b = torch.nn.functional.pad(b, (0, -b.shape[-1] % 8)).unflatten(-1, (-1, 8))
    return (b << torch.arange(8, device=DEV, dtype=torch.uint8)).sum(-1, dtype=torch.uint8)


def _quantize(gen, shape, bits, rotation, sketch):
    """Packed rows of random vectors [B, H, N, D]: codes and norms, with ``sketch`` signs and residual norms too."""
    centers, mid = (torch.from_numpy(t).to(DEV) for t in _codebook(bits, D))
    u = torch.randn(*shape, D, generator=gen, device=DEV)
    u /= u.norm(dim=-1, keepdim=True)
    norms = torch.exp(math.log(20.0) + 0.3 * torch.randn(*shape, generator=gen, device=DEV)).half()
    z = u @ rotation.T
    codes = torch.bucketize(z, mid, out_int32=True)
    out = {"c": _pack(codes.to(torch.uint8), bits), "n": norms}
    if sketch is not None:
        r = u - centers[codes] @ rotation
        out["s"] = _pack((r @ sketch.T >= 0).to(torch.uint8), 1)
        out["r"] = (norms.float() * r.norm(dim=-1)).half()
    return out


def _parents(c, seed):
    """[T] parents of the drafted tokens: -1 for those that follow the history itself."""
    if c["shape"] == "chain":
        p = list(range(-1, c["T"] - 1))
    else:  # breadth first: up to 4 first tokens, a token's children behind its own level
        rng = np.random.default_rng(seed)
        p = [-1 if i < min(4, (c["T"] + 1) // 2) else int(rng.integers(max(0, (i - 4) // 2), i)) for i in range(c["T"])]
    return torch.tensor(p, dtype=torch.int32, device=DEV)


def _prepare_tree(c, seed):
    gen = _gen(seed)
    key_bits = c["bits"] - 1 if c["qjl"] else c["bits"]
    rk, rv = (torch.linalg.qr(torch.randn(D, D, generator=gen, device=DEV)).Q.contiguous() for _ in range(2))
    sketch = torch.randn(D, D, generator=gen, device=DEV) if c["qjl"] else None
    shape = (c["B"], c["Hkv"], c["N"] + c["T"])
    s = {"k": _quantize(gen, shape, key_bits, rk, sketch), "v": _quantize(gen, shape, c["bits"], rv, None), "rk": rk,
         "rv": rv, "sketch": sketch, "kb": key_bits, "vb": c["bits"]}
    for w, bits in (("ck", key_bits), ("cv", c["bits"])):
        s[w] = torch.from_numpy(_codebook(bits, D)[0]).to(DEV)
        s["mid" + w] = torch.from_numpy(_codebook(bits, D)[1]).to(DEV)
    s["q"] = torch.randn(c["B"], c["T"], c["Hq"], D, generator=gen, device=DEV).bfloat16().transpose(1, 2)
    s["parents"] = _parents(c, seed)
    s["starts"] = s["lens"] = None
    if c["ragged"]:  # [start, end) of each sequence's history; its drafted tokens follow at the end
        i = np.arange(c["B"])
        s["starts"] = torch.tensor((7 * i * c["N"]) // 64, dtype=torch.int32, device=DEV)
        s["lens"] = torch.tensor(c["N"] - (5 * i * c["N"]) // 64, dtype=torch.int32, device=DEV)
    if own:  # the handles a program keeps with its layer
        from turboquant.runtime.kernels import CodecParams

        s["key"] = CodecParams(key_bits, rk, s["ck"], s["midck"])
        s["value"] = CodecParams(c["bits"], rv, s["cv"], s["midcv"])
    return s


def _row_bytes(c):
    """Row bytes of a layer's byte buffers (codes and signs), and how many fp16 buffers stand beside them."""
    groups = [(D - c["split"], c["bits"])] + ([(c["split"], c["bits"] + 1)] if c["split"] else [])
    rows = [(d * (b - 1 if c["qjl"] else b) + 7) // 8 for d, b in groups] + [(d * b + 7) // 8 for d, b in groups]
    rows += [(d + 7) // 8 for d, _ in groups] if c["qjl"] else []
    return rows, len(rows)


def _prepare_moves(c, seed):
    gen = _gen(seed)
    tokens = c["N"] + c["T"]
    cap = tokens + 64  # slots in reserve, as a layer keeps them
    rows, halves = _row_bytes(c)
    at = (c["B"], c["Hkv"], cap)
    s = {"buffers": [torch.randint(0, 256, (*at, r), generator=gen, device=DEV, dtype=torch.uint8) for r in rows]
         + [(20.0 * torch.exp(0.3 * torch.randn(at, generator=gen, device=DEV))).half() for _ in range(halves)]}
    rng = np.random.default_rng(seed)
    s["rows"] = s["index"] = None
    if c["op"] == "keep":
        # an accepted path: its first token the likeliest, the later ones from deeper levels
        late = np.sort(rng.choice(np.arange(c["keep"], c["T"]), c["keep"] - 1, replace=False))
        s["index"] = torch.tensor([0, *late], dtype=torch.int32, device=DEV)
    elif c["keep"]:
        score = torch.rand(c["B"], c["Hkv"], tokens, generator=gen, device=DEV)
        s["index"] = score.topk(c["keep"], dim=-1).indices.sort(-1).values.int()
    else:
        s["rows"] = torch.tensor(rng.integers(0, c["B"], c["rows"]), dtype=torch.int32, device=DEV)
    return s


def prepare(case, seed):
    make = {"prompt": _prepare_prompt, "tree": _prepare_tree}.get(case["op"], _prepare_moves)
    return dict(make(case, seed), case=case)


# ---------------------------------------------------------------- one pass


def _plain_prompt(s):
    q, k, v = s["q"].float(), s["k"].float(), s["v"].float()
    B, Hq, S, _ = q.shape
    Hkv = k.shape[1]
    i = torch.arange(S, device=DEV)
    seen = (i[None, :] <= i[:, None])[None]
    if "cu_seqlens" in s:  # the sequence of each row; rows behind the last one belong to none
        seq = torch.bucketize(i, s["cu_seqlens"][1:], right=True, out_int32=True)
        live = seq < s["cu_seqlens"].numel() - 1
        seen = (seen & (seq[None, :] == seq[:, None]) & live[:, None])
    elif "seq_starts" in s:
        ok = i[None, :] >= s["seq_starts"][:, None]
        seen = seen & ok[:, None, :] & ok[:, :, None]
    # each KV head's query heads as rows of one product
    logits = q.reshape(B, Hkv, -1, D) @ k.transpose(-1, -2)
    logits = logits.view(B, Hkv, Hq // Hkv, S, S).mul_(1.0 / math.sqrt(D))
    logits.masked_fill_(~seen[:, None, None], float("-inf"))
    top = logits.amax(-1, keepdim=True)
    p = logits.sub_(torch.where(top == float("-inf"), 0.0, top)).exp_()
    total = p.sum(-1).clamp(min=1e-30)
    out = (p.view(B, Hkv, -1, S) @ v).view(B, Hkv, Hq // Hkv, S, D) / total[..., None]
    return out.view(B, Hq, S, D).to(s["q"].dtype)


def _unpack(rows, bits, n):
    at = torch.arange(n, device=DEV) * bits
    wide = torch.nn.functional.pad(rows, (0, 1)).int()
    return ((wide[..., at // 8] | (wide[..., at // 8 + 1] << 8)) >> (at % 8)) & ((1 << bits) - 1)


def _tree_sees(parents, T):
    """[T, T]: whether node j is node i itself or one of its ancestors."""
    sees = torch.eye(T, dtype=torch.float32, device=DEV)
    child = (parents[:, None] == torch.arange(T, device=DEV)[None, :]).float()  # i's parent is j
    reach = sees + child
    # paths of up to T steps by squaring
    power = functools.reduce(lambda m, _: ((m @ m) > 0).float(), range(max(1, math.ceil(math.log2(T + 1)))), reach)
    return power > 0


def _plain_tree(s):
    c, q = s["case"], s["q"].float()
    B, Hq, T, _ = q.shape
    Hkv, g, n = c["Hkv"], c["Hq"] // c["Hkv"], c["N"] + c["T"]
    keys = (s["ck"][_unpack(s["k"]["c"], s["kb"], D)] @ s["rk"]) * s["k"]["n"].float()[..., None]
    if s["sketch"] is not None:
        pm = 2.0 * _unpack(s["k"]["s"], 1, D).float() - 1.0
        keys += (pm @ s["sketch"]) * (s["k"]["r"].float()[..., None] * (math.sqrt(math.pi / 2) / D))
    values = (s["cv"][_unpack(s["v"]["c"], s["vb"], D)] @ s["rv"]) * s["v"]["n"].float()[..., None]
    slot = torch.arange(n, device=DEV)[None, :]
    first = torch.zeros(B, 1, device=DEV) if s["starts"] is None else s["starts"][:, None]
    end = torch.full((B, 1), c["N"], device=DEV) if s["lens"] is None else s["lens"][:, None].long()
    node = slot - end  # a slot's node, from 0
    sees = _tree_sees(s["parents"], T)
    seen = sees[:, node.clamp(0, T - 1)].transpose(0, 1) & ((node >= 0) & (node < T))[:, None]
    seen |= ((slot >= first) & (slot < end))[:, None]
    logits = (q.reshape(B, Hkv, -1, D) @ keys.transpose(-1, -2)).view(B, Hkv, g, T, n) / math.sqrt(D)
    p = _softmax(logits, seen[:, None, None])
    return (p.view(B, Hkv, -1, n) @ values).view(B, Hq, T, D).to(s["q"].dtype)


def _softmax(logits, seen):
    logits = logits.masked_fill(~seen, float("-inf"))
    p = (logits - logits.amax(-1, keepdim=True)).exp()
    return p / p.sum(-1, keepdim=True)


def _plain_keep(s):
    c, index = s["case"], s["index"].long() + s["case"]["N"]
    [b[:, :, c["N"]:c["N"] + c["keep"]].copy_(b[:, :, index]) for b in s["buffers"]]
    return [b[:, :, c["N"]:c["N"] + c["keep"]] for b in s["buffers"]]


def _plain_gather(s):
    c = s["case"]
    if s["rows"] is not None:
        take = lambda b: b[s["rows"].long(), :, :c["N"]]  # noqa: E731
    else:
        index = s["index"].long()
        heads = torch.arange(c["B"] * c["Hkv"], device=DEV).view(c["B"], c["Hkv"], 1)
        take = lambda b: b.flatten(0, 1)[heads, index]  # noqa: E731
    return [take(b) for b in s["buffers"]]


def run(state):
    s, op = state, state["case"]["op"]
    if not own:
        return {"prompt": _plain_prompt, "tree": _plain_tree, "keep": _plain_keep, "gather": _plain_gather}[op](s)
    from turboquant.runtime import kernels as K
    from turboquant.runtime import prompt_attention

    c = s["case"]
    if op == "prompt":
        return prompt_attention(s["q"], s["k"], s["v"], cu_seqlens=s.get("cu_seqlens"), seq_starts=s.get("seq_starts"))
    if op == "tree":
        return K.tree_attention(s["q"], s["parents"], k_codes=s["k"]["c"], k_norms=s["k"]["n"], v_codes=s["v"]["c"],
                                v_norms=s["v"]["n"], n_tokens=c["N"] + c["T"], key=s["key"], value=s["value"],
                                k_signs=s["k"].get("s"), k_rnorms=s["k"].get("r"), qjl=s["sketch"],
                                seq_starts=s["starts"], seq_lens=s["lens"])
    if op == "keep":
        K.keep_tokens(s["buffers"], s["index"], first=c["N"], tokens=c["T"])
        return [b[:, :, c["N"]:c["N"] + c["keep"]] for b in s["buffers"]]
    return K.gather_tokens(s["buffers"], tokens=c["N"], rows=s["rows"], index=s["index"])


# ---------------------------------------------------------------- what a pass cannot do without


def work(case):
    c = case
    if c["op"] == "prompt":
        lens = _lens(c)
        return {"bytes": sum(lens) * (2 * c["Hq"] + 2 * c["Hkv"]) * D * 2,
                "flops": sum(n * (n + 1) // 2 for n in lens) * c["Hq"] * 4 * D}
    if c["op"] == "tree":
        kb = c["bits"] - 1 if c["qjl"] else c["bits"]
        per = D * (kb + c["bits"] + c["qjl"]) // 8 + 2 * (2 + c["qjl"])
        i = np.arange(c["B"])
        spans = c["N"] - ((7 * i * c["N"]) // 64 + (5 * i * c["N"]) // 64 if c["ragged"] else 0 * i) + c["T"]
        mats = (3 if c["qjl"] else 2) * D * D * 4
        tokens = int(spans.sum())
        return {"bytes": tokens * c["Hkv"] * per + 2 * c["B"] * c["Hq"] * c["T"] * D * 2 + mats,
                "flops": tokens * c["Hq"] * c["T"] * (6 if c["qjl"] else 4) * D}
    rows, halves = _row_bytes(c)
    per = sum(rows) + 2 * halves
    if c["keep"]:
        tokens = 2 * c["keep"] * c["B"]
    else:  # a batch row chosen twice is read once
        tokens = c["N"] * (c["rows"] + min(c["rows"], c["B"]))
    return {"bytes": tokens * c["Hkv"] * per, "flops": 0}


# ---------------------------------------------------------------- the same in 64 bits


def _exact_prompt(c, s):
    lens, (B, Hq, S, _) = _lens(c), s["q"].shape
    out = torch.zeros(B, Hq, S, D, dtype=torch.float64, device=DEV)
    at = 0
    for n, length in enumerate(lens):
        b, a = (0, at) if c["packed"] else (n, S - length)
        at += length
        for h in range(Hq):
            k, v = (s[w][b, h * c["Hkv"] // Hq, a:a + length].double() for w in "kv")
            for i in range(0, length, 4096):
                e = min(i + 4096, length)
                x = s["q"][b, h, a + i:a + e].double() @ k[:e].T / math.sqrt(D)
                x = x.masked_fill(torch.ones_like(x, dtype=torch.bool).triu(i + 1), float("-inf"))
                out[b, h, a + i:a + e] = torch.softmax(x, -1) @ v[:e]
    return out


def _exact_rows(packed, b, h, bits, centers, rotation, sketch):
    """One head's vectors in 64 bits, from its bit streams."""
    def numbers(rows, width):
        bit = np.unpackbits(rows.cpu().numpy(), axis=-1, bitorder="little")[:, :D * width].reshape(-1, D, width)
        return torch.from_numpy((bit.astype(np.int64) << np.arange(width)).sum(-1)).to(DEV)

    x = centers.double()[numbers(packed["c"][b, h], bits)] @ rotation.double() * packed["n"][b, h].double()[:, None]
    if sketch is not None:
        sign = torch.where(numbers(packed["s"][b, h], 1) == 1, 1.0, -1.0).double()
        x = x + math.sqrt(math.pi / 2) / D * packed["r"][b, h].double()[:, None] * (sign @ sketch.double())
    return x


def _exact_tree(c, s):
    parents, g = s["parents"].tolist(), c["Hq"] // c["Hkv"]
    out = torch.empty(c["B"], c["Hq"], c["T"], D, dtype=torch.float64, device=DEV)
    paths = []
    for i in range(c["T"]):
        paths.append([i] + (paths[parents[i]] if parents[i] >= 0 else []))
    for b in range(c["B"]):
        lo = 0 if s["starts"] is None else int(s["starts"][b])
        hi = c["N"] if s["lens"] is None else int(s["lens"][b])
        seen = torch.zeros(c["T"], c["N"] + c["T"], dtype=torch.bool)
        seen[:, lo:hi] = True
        for i, path in enumerate(paths):
            seen[i, [hi + j for j in path]] = True
        for h in range(c["Hkv"]):
            k = _exact_rows(s["k"], b, h, s["kb"], s["ck"], s["rk"], s["sketch"])
            v = _exact_rows(s["v"], b, h, s["vb"], s["cv"], s["rv"], None)
            x = s["q"][b, h * g:(h + 1) * g].double() @ k.T / math.sqrt(D)
            out[b, h * g:(h + 1) * g] = torch.softmax(x.masked_fill(~seen.to(DEV), float("-inf")), -1) @ v
    return out


def _exact_moves(c, s):
    """The norms' values, gathered on the host; codes are bytes."""
    out = []
    for buf in s["buffers"]:
        if buf.dtype == torch.uint8:
            out.append(None)
            continue
        x = buf.cpu().numpy().astype(np.float64)
        if c["op"] == "keep":
            y = x[:, :, c["N"] + s["index"].cpu().numpy()]
        elif s["rows"] is not None:
            y = x[s["rows"].cpu().numpy(), :, :c["N"]]
        else:
            y = np.take_along_axis(x, s["index"].cpu().numpy().astype(np.int64), axis=2)
        out.append(torch.from_numpy(y))
    return out


def exact(case, seed):
    s = prepare(case, seed)
    return {"prompt": _exact_prompt, "tree": _exact_tree}.get(case["op"], _exact_moves)(case, s)
