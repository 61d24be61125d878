"""Timing cases of the operators for prompts that many sequences share, and for long histories read in part.

* ``prefix``  attention of one query token per sequence where several sequences continue one packed prompt: the prompt
              is stored and read once for all of them, each has packed tokens of its own behind it
              (``turboquant.runtime.kernels.prefix_attention``);
* ``bounds``  the elementwise least and largest key of every 64 tokens, rounded outward to 8 bits
              (``turboquant.runtime.kernels.block_bounds``);
* ``select``  the blocks of 64 tokens that a query may give the largest logits, from those bounds
              (``turboquant.runtime.kernels.select_blocks``);
* ``blocks``  attention of one query token per sequence over chosen blocks of a packed cache
              (``turboquant.runtime.kernels.block_attention``).

Head dimension 128 throughout.  Queries are N(0, 1); keys and values have iid N(0, 1) directions, packed ones with
lognormal norms around 20.  Keys that are bounded have, beside that, channels with a mean of their own and a drift
along the text, as keys behind a position rotation do.  Packed caches are quantized here with elementary operations: a
random rotation, Lloyd-Max codes of a coordinate, fp16 norms and, with QJL, the signs of a Gaussian sketch of the
key's residual and its fp16 norm.
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
BLOCK = 64  # tokens of a block
DEV = "cuda"


# ---------------------------------------------------------------- cases


def _prefix(name, counts, Hq, Hkv, N, M, bits, qjl, dtype="bf16", ragged=False):
    """``counts`` as text: how many sequences continue each prompt of N tokens; up to M own tokens for each."""
    c = {"op": "prefix", "counts": counts, "Hq": Hq, "Hkv": Hkv, "N": N, "M": M, "bits": bits, "qjl": qjl, "dtype": dtype,
         "ragged": ragged}
    return dict(c, name=name) if name else c


def _bounds(name, B, Hkv, T, first):
    c = {"op": "bounds", "B": B, "Hkv": Hkv, "T": T, "first": first}
    return dict(c, name=name) if name else c


def _select(name, B, Hq, Hkv, N, keep, sink, recent, dtype="bf16", ragged=False):
    c = {"op": "select", "B": B, "Hq": Hq, "Hkv": Hkv, "N": N, "keep": keep, "sink": sink, "recent": recent, "dtype": dtype,
         "ragged": ragged}
    return dict(c, name=name) if name else c


def _blocks(name, B, Hq, Hkv, N, keep, bits, qjl, ragged=False):
    c = {"op": "blocks", "B": B, "Hq": Hq, "Hkv": Hkv, "N": N, "keep": keep, "bits": bits, "qjl": qjl, "ragged": ragged}
    return dict(c, name=name) if name else c


def listed():
    return [
        # two answers to one short chat, some tokens into them: the smallest, latency counts
        _prefix("prefix_pair", "2", 32, 8, 1037, 19, 4, True),
        # 8 beams for each of 4 padded prompts, beams of a few to 64 tokens; a fp16 model's 3-bit Q_mse cache
        _prefix("prefix_beams", "8 8 8 8", 28, 4, 8192, 64, 3, False, dtype="fp16", ragged=True),
        # a serving batch behind one system prompt of 32K
        _prefix("prefix_batch_32k", "32", 32, 8, 32768, 256, 4, True),
        # three documents with as many readers as come, 40/8 heads, 128K tokens each: the largest
        _prefix("prefix_readers_131k", "21 3 8", 40, 8, 131072, 1024, 4, True),
        # one block filled in each of 8 sequences: latency counts
        _bounds("bounds_step", 8, 8, 64, 511),
        # a batch of prompts of 32K, the last block of each not full
        _bounds("bounds_prompts_32k", 8, 8, 32749, 0),
        # 32 of the 129 blocks of a chat
        _select("select_chat", 1, 32, 8, 8195, 32, 1, 2),
        # a batch at 32K, 64 blocks each; sequences with ranges of their own
        _select("select_8b_32k", 8, 32, 8, 32768, 64, 1, 2, ragged=True),
        # four long documents, 128 of 2048 blocks each; 5 query heads per KV head of a fp16 model
        _select("select_131k", 4, 40, 8, 131072, 128, 1, 2, dtype="fp16"),
        # the chat's chosen blocks
        _blocks("blocks_chat", 1, 32, 8, 8195, 32, 4, True),
        # the batch's chosen blocks
        _blocks("blocks_8b_32k", 8, 32, 8, 32768, 64, 4, True, ragged=True),
        # the documents' chosen blocks, 3-bit Q_mse, 7 query heads per KV head
        _blocks("blocks_131k", 16, 28, 4, 131072, 128, 3, False),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("prefix", "prefix", "prefix", "bounds", "select", "select", "blocks", "blocks"))
    Hkv, g = rng.choice(((8, 4), (4, 7), (8, 5), (2, 8), (4, 1), (8, 2)))
    qjl = rng.random() < 0.6
    bits = rng.choice((3, 4, 4)) if qjl else rng.choice((2, 3, 4))
    if op == "prefix":
        counts = [_log(rng, 1, 32)] if rng.random() < 0.4 else [_log(rng, 1, 12) for _ in range(rng.randint(2, 4))]
        return _prefix(None, " ".join(map(str, counts)), Hkv * g, Hkv, _log(rng, 64, 32768), _log(rng, 1, 512), bits, qjl,
                       rng.choice(("bf16", "bf16", "fp16")), rng.random() < 0.4)
    if op == "bounds":
        return _bounds(None, rng.choice((1, 2, 4)), Hkv, _log(rng, 1, 32768), rng.randint(0, 300))
    B, N = rng.choice((1, 2, 3, 4)), _log(rng, 600, 65536)
    keep = max(4, min(_log(rng, 4, 128), N // BLOCK // 2))
    if op == "select":
        return _select(None, B, Hkv * g, Hkv, N, keep, rng.randint(0, 1), rng.randint(1, 2), rng.choice(("bf16", "bf16", "fp16")),
                       rng.random() < 0.4)
    return _blocks(None, B, Hkv * g, Hkv, N, keep, bits, qjl, rng.random() < 0.4)


# ---------------------------------------------------------------- preparing


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _dtype(c):
    return torch.float16 if c.get("dtype") == "fp16" else torch.bfloat16


def _counts(c):
    return [int(x) for x in c["counts"].split()]


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


def _quantize_rows(gen, shape, bits, rotation, sketch):
    centers, mid = (torch.from_numpy(t).to(DEV) for t in _codebook(bits, D))
    u = torch.randn(*shape, D, generator=gen, device=DEV)
    u /= u.norm(dim=-1, keepdim=True)
    norms = torch.exp(math.log(20.0) + 0.3 * torch.randn(*shape, generator=gen, device=DEV)).half()
    codes = torch.bucketize(u @ rotation.T, mid, out_int32=True)
    out = {"k_codes": _pack(codes.to(torch.uint8), bits), "k_norms": norms}
    if sketch is not None:
        r = u - centers[codes] @ rotation
        out["k_signs"] = _pack((r @ sketch.T >= 0).to(torch.uint8), 1)
        out["k_rnorms"] = (norms.float() * r.norm(dim=-1)).half()
    return out


def _quantize(gen, rows, heads, tokens, codec):
    """A packed cache [rows, heads, tokens, ...] of random vectors, a row at a time."""
    made = []
    for _ in range(rows):
        one = _quantize_rows(gen, (heads, tokens), codec["kb"], codec["rk"], codec["sketch"])
        v = _quantize_rows(gen, (heads, tokens), codec["vb"], codec["rv"], None)
        made.append(dict(one, v_codes=v["k_codes"], v_norms=v["k_norms"]))
    return {name: torch.stack([m[name] for m in made]) for name in made[0]}


def _codec(c, gen):
    """The layer's rotations, codebooks and sketch, and the package's handles on them."""
    kb = c["bits"] - 1 if c["qjl"] else c["bits"]
    rk, rv = (torch.linalg.qr(torch.randn(D, D, generator=gen, device=DEV)).Q.contiguous() for _ in range(2))
    s = {"kb": kb, "vb": c["bits"], "rk": rk, "rv": rv,
         "sketch": torch.randn(D, D, generator=gen, device=DEV) if c["qjl"] else None}
    for w, bits in (("ck", kb), ("cv", c["bits"])):
        s[w], s["mid" + w] = (torch.from_numpy(t).to(DEV) for t in _codebook(bits, D))
    if own:  # the handles a program keeps with its layer
        from turboquant.runtime.kernels import CodecParams

        s["key"] = CodecParams(kb, rk, s["ck"], s["midck"])
        s["value"] = CodecParams(c["bits"], rv, s["cv"], s["midcv"])
    return s


def _query(gen, B, Hq, dtype):
    """A projection's output for one token per sequence."""
    return torch.randn(B, 1, Hq, D, generator=gen, device=DEV).to(dtype).transpose(1, 2)


def _prepare_prefix(c, seed):
    gen, counts = _gen(seed), _counts(c)
    P, B, most = len(counts), sum(counts), max(counts)
    codec = _codec(c, gen)
    s = {"codec": codec, "prefix": _quantize(gen, P, c["Hkv"], c["N"], codec),
         "own": _quantize(gen, B, c["Hkv"], c["M"], codec), "q": _query(gen, B, c["Hq"], _dtype(c))}
    # the prompts' first rows among the sequences, needed where they have different numbers of them
    s["cu_rows"] = torch.tensor(np.cumsum([0] + counts), dtype=torch.int32, device=DEV) if len(set(counts)) > 1 else None
    s["max_rows"] = most
    s["starts"] = s["lens"] = None
    if c["ragged"]:  # left padding of the prompts, and as many own tokens as each sequence has so far (some none)
        p, b = np.arange(P), np.arange(B)
        s["starts"] = torch.tensor((5 * p * c["N"]) // 64, dtype=torch.int32, device=DEV)
        s["lens"] = torch.tensor((b * 37 + c["M"]) % (c["M"] + 1), dtype=torch.int32, device=DEV)
    # where a sequence stands among [prompts, most sequences of one], and who stands there
    place = np.concatenate([np.arange(n) + i * most for i, n in enumerate(counts)])
    who = np.zeros(P * most, np.int64)
    who[place] = np.arange(B)
    s["place"], s["who"] = torch.from_numpy(place).to(DEV), torch.from_numpy(who).to(DEV).view(P, most)
    return s


def _keys(gen, B, Hkv, T, seed):
    """bf16 keys [B, Hkv, T, D] as a projection and a rotation leave them, token by token in memory."""
    x = torch.randn(B, T, Hkv, D, generator=gen, device=DEV)
    rate = 2.0 ** -torch.linspace(0, 14, D, device=DEV)
    at = torch.arange(T, device=DEV, dtype=torch.float32)[:, None] * rate + seed % 7
    x += 2.0 * torch.randn(1, 1, Hkv, D, generator=gen, device=DEV) * torch.cos(at)[None, :, None]
    return (x * 1.4).bfloat16().transpose(1, 2)


def _prepare_bounds(c, seed):
    n = -(-c["T"] // BLOCK)
    cap = c["first"] + n + 4  # a layer keeps places in reserve
    return {"k": _keys(_gen(seed), c["B"], c["Hkv"], c["T"], seed), "n": n,
            "lohi": torch.zeros(c["B"], c["Hkv"], cap, 2, D, dtype=torch.int8, device=DEV),
            "scale": torch.ones(c["B"], c["Hkv"], cap, device=DEV)}


def _ranges(c):
    """[start, end) of each sequence of a ragged batch."""
    i = np.arange(c["B"])
    starts, ends = (3 * i * c["N"]) // 64, c["N"] - (2 * i * c["N"]) // 64
    return (torch.tensor(x, dtype=torch.int32, device=DEV) for x in (starts, ends))


def _prepare_select(c, seed):
    gen = _gen(seed)
    n = -(-c["N"] // BLOCK)
    s = {"lohi": torch.empty(c["B"], c["Hkv"], n, 2, D, dtype=torch.int8, device=DEV),
         "scale": torch.empty(c["B"], c["Hkv"], n, device=DEV), "q": _query(gen, c["B"], c["Hq"], _dtype(c))}
    for b in range(c["B"]):
        lohi, scale = _plain_bounds(_keys(gen, 1, c["Hkv"], c["N"], seed + b))
        s["lohi"][b], s["scale"][b] = lohi[0], scale[0]
    s["starts"], s["lens"] = _ranges(c) if c["ragged"] else (None, None)
    return s


def _prepare_blocks(c, seed):
    gen = _gen(seed)
    codec = _codec(c, gen)
    s = {"codec": codec, "cache": _quantize(gen, c["B"], c["Hkv"], c["N"], codec),
         "q": _query(gen, c["B"], c["Hq"], torch.bfloat16)}
    n = -(-c["N"] // BLOCK)
    # the first block, the last two and the likeliest of the others, in order
    score = torch.rand(c["B"], c["Hkv"], n, generator=gen, device=DEV)
    score[..., :1], score[..., -2:] = 2.0, 2.0
    s["starts"], s["lens"] = _ranges(c) if c["ragged"] else (None, None)
    if c["ragged"]:  # blocks outside a sequence's range are not chosen; a short range leaves places empty
        at = torch.arange(n, device=DEV) * BLOCK
        score[((at + BLOCK <= s["starts"][:, None]) | (at >= s["lens"][:, None]))[:, None].expand_as(score)] = -1.0
    top = score.sort(dim=-1, descending=True, stable=True)
    s["blocks"] = torch.where(top.values >= 0, top.indices, n + 1)[..., :c["keep"]].sort(-1).values.int()
    s["blocks"][s["blocks"] > n] = -1
    return s


def prepare(case, seed):
    make = {"prefix": _prepare_prefix, "bounds": _prepare_bounds, "select": _prepare_select, "blocks": _prepare_blocks}
    return dict(make[case["op"]](case, seed), case=case)


# ---------------------------------------------------------------- one pass


def _unpack(rows, bits, n):
    at = torch.arange(n, device=DEV) * bits
    wide = torch.nn.functional.pad(rows, (0, 1)).int()
    return ((wide[..., at // 8] | (wide[..., at // 8 + 1] << 8)) >> (at % 8)) & ((1 << bits) - 1)


def _rows(t, x):
    """fp32 keys and values of packed rows ``t`` under the codec ``x``."""
    keys = (x["ck"][_unpack(t["k_codes"], x["kb"], D)] @ x["rk"]) * t["k_norms"].float()[..., None]
    if x["sketch"] is not None:
        pm = 2.0 * _unpack(t["k_signs"], 1, D).float() - 1.0
        keys += (pm @ x["sketch"]) * (t["k_rnorms"].float()[..., None] * (math.sqrt(math.pi / 2) / D))
    return keys, (x["cv"][_unpack(t["v_codes"], x["vb"], D)] @ x["rv"]) * t["v_norms"].float()[..., None]


def _softmax(logits):
    top = logits.amax(-1, keepdim=True)
    p = (logits - torch.where(top == float("-inf"), 0.0, top)).exp_()
    return p / p.sum(-1, keepdim=True).clamp(min=1e-30)


def _plain_prefix(s):
    c, x = s["case"], s["codec"]
    (P, most), Hkv, g = s["who"].shape, c["Hkv"], c["Hq"] // c["Hkv"]
    q = s["q"].float().view(-1, Hkv, g, D) / math.sqrt(D)
    keys, values = _rows(s["prefix"], x)
    mine, my_values = _rows(s["own"], x)
    rows = q[s["who"]].transpose(1, 2).reshape(P, Hkv, most * g, D)  # every prompt's queries as rows of one product
    logits = (rows @ keys.transpose(-1, -2)).view(P, Hkv, most, g, c["N"])
    if s["starts"] is not None:
        behind = torch.arange(c["N"], device=DEV) >= s["starts"][:, None]
        logits = logits.masked_fill(~behind[:, None, None, None], float("-inf"))
    more = q @ mine.transpose(-1, -2)
    if s["lens"] is not None:
        there = torch.arange(c["M"], device=DEV) < s["lens"][:, None]
        more = more.masked_fill(~there[:, None, None], float("-inf"))
    p = _softmax(torch.cat((logits, more[s["who"]].transpose(1, 2)), -1))
    out = (p[..., :c["N"]].reshape(P, Hkv, most * g, c["N"]) @ values).view(P, Hkv, most, g, D)
    out = out.transpose(1, 2).flatten(0, 1)[s["place"]]
    out += p[..., c["N"]:].transpose(1, 2).flatten(0, 1)[s["place"]] @ my_values
    return out.view(-1, c["Hq"], D).to(s["q"].dtype)


def _steps(most):
    """The least power of two whose 127-fold is not below ``most``, from 2^-100 to 2^100."""
    m, e = torch.frexp(most)
    e = torch.where(most > 0, torch.where(m > 127 / 128, e - 6, e - 7), -100).clamp(-100, 100)
    return ((e + 127) << 23).int().view(torch.float32)


def _plain_bounds(k):
    """Bounds of every BLOCK tokens of k [B, H, T, D]: whole numbers [B, H, n, 2, D], and what one of them stands for."""
    T = k.shape[2]
    at = torch.arange(-(-T // BLOCK) * BLOCK, device=DEV).clamp(max=T - 1)  # a block that is not full: its last token again
    k = k.float()[:, :, at].unflatten(2, (-1, BLOCK))
    lo, hi = k.amin(3), k.amax(3)
    scale = _steps(torch.maximum(-lo, hi).amax(-1))
    lohi = torch.stack(((lo / scale[..., None]).floor(), (hi / scale[..., None]).ceil()), -2)
    return lohi.clamp(-127, 127).to(torch.int8), scale


def _plain_bounds_into(s):
    c = s["case"]
    to = slice(c["first"], c["first"] + s["n"])
    s["lohi"][:, :, to], s["scale"][:, :, to] = _plain_bounds(s["k"])
    return s["lohi"][:, :, to] * s["scale"][:, :, to, None, None]


def _plain_select(s):
    c, n = s["case"], s["lohi"].shape[2]
    q = s["q"].float().view(c["B"], c["Hkv"], -1, D)
    x = (q / _steps(q.abs().amax((-1, -2)))[..., None, None]).round().clamp(-127, 127)
    lo, hi = s["lohi"].float().unbind(-2)
    most = x.clamp(min=0) @ hi.transpose(-1, -2) + x.clamp(max=0) @ lo.transpose(-1, -2)  # whole numbers below 2^24
    score = most.amax(2) * s["scale"]
    j = torch.arange(n, device=DEV)
    first = torch.zeros(c["B"], 1, device=DEV) if s["starts"] is None else s["starts"][:, None] // BLOCK
    last = torch.full((c["B"], 1), n, device=DEV) if s["lens"] is None else (s["lens"][:, None] + BLOCK - 1) // BLOCK
    always = (j < first + c["sink"]) | (j >= last - c["recent"])
    score = torch.where(always[:, None], float("inf"), score)
    score = torch.where(((j >= first) & (j < last))[:, None], score, float("-inf"))
    top = score.sort(dim=-1, descending=True, stable=True)
    chosen = torch.where(top.values > float("-inf"), top.indices, n)[..., :c["keep"]].sort(-1).values
    return torch.where(chosen < n, chosen, -1).int()


def _plain_blocks(s):
    c, x, b = s["case"], s["codec"], s["blocks"].long()
    Hkv = c["Hkv"]
    token = (b[..., None] * BLOCK + torch.arange(BLOCK, device=DEV)).flatten(-2)  # [B, Hkv, keep * BLOCK]
    seen = (b >= 0).repeat_interleave(BLOCK, -1) & (token < c["N"])
    if s["starts"] is not None:
        seen &= (token >= s["starts"][:, None, None]) & (token < s["lens"][:, None, None])
    at = token.clamp(0, c["N"] - 1) + torch.arange(c["B"] * Hkv, device=DEV).view(c["B"], Hkv, 1) * c["N"]
    keys, values = _rows({w: t.flatten(0, 2)[at] for w, t in s["cache"].items()}, x)
    logits = s["q"].float().view(c["B"], Hkv, -1, D) @ keys.transpose(-1, -2) / math.sqrt(D)
    p = _softmax(logits.masked_fill(~seen[:, :, None], float("-inf")))
    return (p @ values).view(c["B"], c["Hq"], D).to(s["q"].dtype)


def run(state):
    s, c = state, state["case"]
    if not own:
        return {"prefix": _plain_prefix, "bounds": _plain_bounds_into, "select": _plain_select, "blocks": _plain_blocks}[c["op"]](s)
    from turboquant.runtime import kernels as K

    if c["op"] == "prefix":
        x = s["codec"]
        return K.prefix_attention(s["q"], s["prefix"], s["own"], n_prefix=c["N"], n_own=c["M"], key=x["key"], value=x["value"],
                                  qjl=x["sketch"], cu_rows=s["cu_rows"], max_rows=s["max_rows"], prefix_starts=s["starts"],
                                  own_lens=s["lens"])
    if c["op"] == "bounds":
        K.block_bounds(s["k"], s["lohi"], s["scale"], first=c["first"])
        to = slice(c["first"], c["first"] + s["n"])
        return s["lohi"][:, :, to] * s["scale"][:, :, to, None, None]
    if c["op"] == "select":
        return K.select_blocks(s["q"], s["lohi"], s["scale"], n_tokens=c["N"], keep=c["keep"], sink=c["sink"], recent=c["recent"],
                               seq_starts=s["starts"], seq_lens=s["lens"])
    x = s["codec"]
    return K.block_attention(s["q"], s["blocks"], **s["cache"], n_tokens=c["N"], key=x["key"], value=x["value"], qjl=x["sketch"],
                             seq_starts=s["starts"], seq_lens=s["lens"])


# ---------------------------------------------------------------- what a pass cannot do without


def _row_bytes(c):
    """Bytes of a token's key and value of one head, and of the layer's matrices."""
    kb = c["bits"] - 1 if c["qjl"] else c["bits"]
    return D * (kb + c["bits"] + c["qjl"]) // 8 + 2 * (2 + c["qjl"]), (3 if c["qjl"] else 2) * D * D * 4


def work(case):
    c = case
    if c["op"] == "bounds":
        tokens, n = c["B"] * c["Hkv"] * c["T"], c["B"] * c["Hkv"] * -(-c["T"] // BLOCK)
        return {"bytes": tokens * D * 2 + n * (2 * D + 4), "flops": 2 * tokens * D}
    i = np.arange(c.get("B", 1))
    lo, hi = ((3 * i * c["N"]) // 64, c["N"] - (2 * i * c["N"]) // 64) if c["ragged"] else (0 * i, c["N"] + 0 * i)
    n = -(-hi // BLOCK) - lo // BLOCK  # blocks of each sequence's range
    if c["op"] == "select":
        scored = int(np.maximum(n - c["sink"] - c["recent"], 0).sum()) * c["Hkv"]
        return {"bytes": scored * (2 * D + 4) + c["B"] * c["Hq"] * D * 2 + c["B"] * c["Hkv"] * c["keep"] * 4,
                "flops": scored * c["Hq"] // c["Hkv"] * 4 * D}
    per, mats = _row_bytes(c)
    ops = (6 if c["qjl"] else 4) * D * c["Hq"]
    if c["op"] == "blocks":
        tokens = int(np.minimum(np.minimum(n, c["keep"]) * BLOCK, hi - lo).sum())
        return {"bytes": tokens * c["Hkv"] * per + c["B"] * (c["Hq"] * D * 4 + c["Hkv"] * c["keep"] * 4) + mats, "flops": tokens * ops}
    counts = _counts(c)
    B, spans = sum(counts), np.array([c["N"] - (5 * p * c["N"] // 64 if c["ragged"] else 0) for p in range(len(counts))])
    mine = int(((np.arange(B) * 37 + c["M"]) % (c["M"] + 1)).sum()) if c["ragged"] else B * c["M"]
    return {"bytes": (int(spans.sum()) + mine) * c["Hkv"] * per + B * c["Hq"] * D * 4 + mats,
            "flops": (int((spans * np.array(counts)).sum()) + mine) * ops}


# ---------------------------------------------------------------- the same in 64 bits


def _exact_codes(rows, bits):
    """Codes of packed rows [n, bytes], from their single bits."""
    bit = (rows[:, :, None] >> torch.arange(8, device=DEV, dtype=torch.uint8)) & 1
    bit = bit.flatten(1)[:, :D * bits].reshape(-1, D, bits).long()
    return sum(bit[..., i] << i for i in range(bits))


def _exact_rows(cache, r, h, x):
    """One head's keys and values of a cache's row in 64 bits."""
    k = x["ck"].double()[_exact_codes(cache["k_codes"][r, h], x["kb"])] @ x["rk"].double()
    k = k * cache["k_norms"][r, h].double()[:, None]
    if x["sketch"] is not None:
        sign = torch.where(_exact_codes(cache["k_signs"][r, h], 1) == 1, 1.0, -1.0).double()
        k = k + math.sqrt(math.pi / 2) / D * cache["k_rnorms"][r, h].double()[:, None] * (sign @ x["sketch"].double())
    v = x["cv"].double()[_exact_codes(cache["v_codes"][r, h], x["vb"])] @ x["rv"].double()
    return k, v * cache["v_norms"][r, h].double()[:, None]


def _exact_prefix(c, s):
    counts, g, x = _counts(c), c["Hq"] // c["Hkv"], s["codec"]
    out = torch.zeros(sum(counts), c["Hq"], D, dtype=torch.float64, device=DEV)
    b = 0
    for p, n in enumerate(counts):
        lo = 0 if s["starts"] is None else int(s["starts"][p])
        for h in range(c["Hkv"]):
            keys, values = (t[lo:] for t in _exact_rows(s["prefix"], p, h, x))
            for i in range(b, b + n):
                m = c["M"] if s["lens"] is None else int(s["lens"][i])
                mine, more = (t[:m] for t in _exact_rows(s["own"], i, h, x))
                k, v = torch.cat((keys, mine)), torch.cat((values, more))
                w = torch.softmax(s["q"][i, h * g:(h + 1) * g, 0].double() @ k.T / math.sqrt(D), -1)
                out[i, h * g:(h + 1) * g] = w @ v
        b += n
    return out


def _exact_steps(most):
    """Powers of two by the definition: 127 of one are not below ``most``, 127 of its half are."""
    e = np.full(most.shape, -100)
    for k in range(-99, 101):
        e[127.0 * 2.0 ** (k - 1) < most] = k
    return 2.0 ** e


def _exact_bounds(k):
    """(whole numbers as doubles [B, H, n, 2, D], steps [B, H, n]) of k [B, H, T, D], on the host."""
    x = k.double().cpu().numpy()
    cut = np.arange(0, x.shape[2], BLOCK)
    lo, hi = np.minimum.reduceat(x, cut, axis=2), np.maximum.reduceat(x, cut, axis=2)
    step = _exact_steps(np.maximum(-lo, hi).max(-1))
    return np.stack((np.floor(lo / step[..., None]), np.ceil(hi / step[..., None])), -2), step


def _exact_select(c, s):
    """The choice, block by block in order of (score, index), on the host."""
    lohi, scale = s["lohi"].cpu().numpy().astype(np.float64), s["scale"].double().cpu().numpy()
    q, g, n = s["q"].double().cpu().numpy()[:, :, 0], c["Hq"] // c["Hkv"], lohi.shape[2]
    out = np.full((c["B"], c["Hkv"], c["keep"]), -1, np.int32)
    for b in range(c["B"]):
        lo = 0 if s["starts"] is None else int(s["starts"][b]) // BLOCK
        hi = n if s["lens"] is None else -(-int(s["lens"][b]) // BLOCK)
        for h in range(c["Hkv"]):
            x = q[b, h * g:(h + 1) * g]
            x = np.clip(np.rint(x / _exact_steps(np.abs(x).max(keepdims=True))), -127, 127)
            most = np.maximum(x[:, None] * lohi[b, h, None, :, 0], x[:, None] * lohi[b, h, None, :, 1]).sum(-1).max(0) * scale[b, h]
            fixed = [j for j in range(lo, hi) if j < lo + c["sink"] or j >= hi - c["recent"]]
            rest = sorted(set(range(lo, hi)) - set(fixed), key=lambda j: (-most[j], j))
            chosen = sorted((fixed + rest)[:c["keep"]])
            out[b, h, :len(chosen)] = chosen
    return torch.from_numpy(out)


def _exact_blocks(c, s):
    g, x = c["Hq"] // c["Hkv"], s["codec"]
    out = torch.zeros(c["B"], c["Hq"], D, dtype=torch.float64, device=DEV)
    for b in range(c["B"]):
        lo, hi = (0, c["N"]) if s["starts"] is None else (int(s["starts"][b]), int(s["lens"][b]))
        for h in range(c["Hkv"]):
            slots = [np.arange(max(j * BLOCK, lo), min((j + 1) * BLOCK, hi)) for j in s["blocks"][b, h].tolist() if j >= 0]
            at = torch.from_numpy(np.concatenate(slots)).to(DEV)
            k, v = _exact_rows({w: t[b:b + 1, h:h + 1, at] for w, t in s["cache"].items()}, 0, 0, x)
            w = torch.softmax(s["q"][b, h * g:(h + 1) * g, 0].double() @ k.T / math.sqrt(D), -1)
            out[b, h * g:(h + 1) * g] = w @ v
    return out


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "bounds":
        lohi, step = _exact_bounds(s["k"])
        return torch.from_numpy(lohi * step[..., None, None])
    return {"prefix": _exact_prefix, "select": _exact_select, "blocks": _exact_blocks}[case["op"]](case, s)
