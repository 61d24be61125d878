"""Packed layers of synthetic keys and values, and their rows and attention in 64 bits."""

import math

import torch

from turboquant.runtime.packed_qmse_cache import PackedMSELayer
from turboquant.runtime.synthetic import kv_bf16

D = 128
BITS = [(4, True), (3, True), (2, True), (4, False), (3, False), (2, False), (1, False)]

#: Queries rotated, and centroids, are rounded to fp16, by at most 2^-11 of each (2.8e-4 root mean square); a logit is a sum of 128
#: products of the two, |q| 11 and |k| about 20: 7e-4, with the QJL part as much again, weights and value centroids 2.8e-4 each.  Of the
#: output's largest element that is 2e-3 at most, the package's tolerance of its other decode kernels; a 16-bit output adds half a step.
TOL = 2e-3


def randn(shape, seed, dtype=torch.bfloat16):
    return torch.randn(shape, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda").to(dtype)


def make_layer(B, Hkv, N, bits, qjl, seed=0, dense=0, **more):
    k, v = kv_bf16((B, Hkv, N + dense, D), seed=seed), kv_bf16((B, Hkv, N + dense, D), seed=seed + 1)
    layer = PackedMSELayer(bits=bits, use_qjl_keys=qjl, quantize_decode=dense == 0, **more)
    layer.initialize_from_dense(k[:, :, :N], v[:, :, :N])
    layer._lazy_update = True
    if dense:
        layer.update(k[:, :, N:], v[:, :, N:])
    return layer


def arrays(layer):
    """The layer's packed arrays by the names the kernels' wrappers take."""
    s = layer._store
    return {"k_codes": s.kc, "k_norms": s.kn, "k_signs": s.ks, "k_rnorms": s.kr, "v_codes": s.vc, "v_norms": s.vn}


def codec(layer):
    c = layer.codecs
    return {"key": c.key, "value": c.value, "qjl": c.qjl}


def _unpack(rows, bits, n):
    at = torch.arange(n, device="cuda") * bits
    wide = torch.nn.functional.pad(rows, (0, 1)).int()
    return (((wide[..., at // 8] | (wide[..., at // 8 + 1] << 8)) >> (at % 8)) & ((1 << bits) - 1)).long()


def rows64(layer):
    """Keys and values [B, H, n, D] of a one-group layer's packed tokens in 64 bits."""
    st, c, n = layer._store, layer.codecs, layer.packed_seq_length()
    k = c.key.centers.double()[_unpack(st.kc[:, :, :n], c.key_bits, D)] @ c.key.rotation.double()
    k = k * st.kn[:, :, :n].double()[..., None]
    if c.qjl is not None:
        pm = 2.0 * _unpack(st.ks[:, :, :n], 1, D).double() - 1.0
        k = k + (pm @ c.qjl.double()) * st.kr[:, :, :n].double()[..., None] * (math.sqrt(math.pi / 2) / D)
    v = c.value.centers.double()[_unpack(st.vc[:, :, :n], c.value_bits, D)] @ c.value.rotation.double()
    return k, v * st.vn[:, :, :n].double()[..., None]


def attend64(q, k, v, mask=None, scale=None):
    """(outputs [B, Hq, D], lse [B, Hq]) of one query a row, q [B, Hq, D], k and v [B, H, n, D], mask bool [B or 1, H or 1, n]; nothing
    attended: 0 and -inf."""
    B, Hq, _ = q.shape
    H, n = k.shape[1:3]
    if n == 0:
        return torch.zeros(B, Hq, D, dtype=torch.float64, device="cuda"), torch.full((B, Hq), -math.inf, device="cuda").double()
    x = (q.double().view(B, H, Hq // H, D) @ k.transpose(-1, -2).contiguous()) * (D ** -0.5 if scale is None else scale)
    if mask is not None:
        x = x.masked_fill(~mask[:, :, None], -math.inf)
    lse = torch.logsumexp(x, -1)
    p = torch.exp(x - torch.where(torch.isfinite(lse), lse, 0.0)[..., None])
    return (p @ v).view(B, Hq, D), lse.view(B, Hq)


def check(got, ref, tol=TOL):
    assert torch.isfinite(got).all()
    half = torch.finfo(got.dtype).eps / 2 if got.dtype != torch.float32 else 0.0
    assert ((got.double() - ref).abs() <= tol * ref.abs().max() + 2 * half * ref.abs()).all()


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")
