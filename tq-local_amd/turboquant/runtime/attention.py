"""TurboQuant attention -- HF Transformers ``AttentionInterface`` backend.

``turboquant_attention_forward`` is registered under the name "turboquant"
(reference ``runtime/attention.py:28-120``).  With a packed cache layer on
the module (``module._tq_cache_layer``) a decode step runs the fused libtq
kernel over the packed history, and several query tokens at once run
``chunked_turboquant_attention`` (libtq decoding, fp32 online softmax); without a
packed layer (prefill, norm-guarded dense layers, layers whose tokens are all
dense) it is plain SDPA, as in the reference.  "turboquant_prompt" is the same with whole causal prompts on libtq's own
kernel (``prompt_attention``); ``tree_attention`` is the call for drafted tokens.

``fused_attention`` replaces the reference's Triton host wrapper
(``runtime/triton_kernels.py:238-368``) with its contract (None = not applicable,
which here means more than one query token, a GQA group wider than 8 query heads
per KV head, or a mask whose attended slots are not contiguous).  Unlike the
reference it accepts any batch size and honours left padding (and right padding
before the packed history ends) from the attention mask.

Outlier-split layers run libtq's channel-group attention kernel
(``tq_decode_attention_groups``), which scores each channel group in its own
rotated space; the reference's fused kernel refuses such layers
(``triton_kernels.py:252-253``) and its chunked path
(``runtime/attention.py:215-304``) dequantises K and V for every step instead.
"""

from __future__ import annotations

import functools
import math
import threading
from typing import TYPE_CHECKING

import torch
import torch.nn.functional as F

from turboquant.runtime import _lib
from turboquant.runtime import kernels as K

if TYPE_CHECKING:
    from turboquant.runtime.packed_qmse_cache import BlockChoice, PackedMSELayer
    from turboquant.runtime.shared_prefix import SharedPrefixLayer


def _attend_mask(attention_mask: torch.Tensor, B: int, total: int) -> torch.Tensor:
    """The decode row of an HF mask as bool [B, total] (True = attend).

    The mask is [B, 1, Sq, kv] (bool, or additive float) or [B, kv]."""
    m = attention_mask
    if m.dim() == 4:
        m = m[:, 0, -1, :]
    if m.dtype != torch.bool:
        m = m > torch.finfo(m.dtype).min / 2 if m.is_floating_point() else m != 0
    m = m[:, :total]
    if m.shape[0] == 1 and B > 1:
        m = m.expand(B, -1)
    return m


#: the ranges of the last mask seen, per host thread (an HF forward hands every layer the same
#: mask tensor): (mask, its version counter, B, total, check, device, stream) -> (starts, ends); holding the mask
#: keeps its memory from being reused by another tensor while the entry is live.  A step on another stream finds its own:
#: it does not wait for this one
_tls = threading.local()


_UNKNOWN_MASK = ("a captured step cannot look whether its mask's rows are ranges of tokens: take the step with the same mask before the "
                 "capture, or set _tq_mask_contiguous of the cache's layers")


def _version(t: torch.Tensor) -> int | None:
    """A tensor's version counter; tensors made in inference mode have none, and nothing is kept for them."""
    return None if t.is_inference() else t._version


def _valid_range(attention_mask: torch.Tensor | None, B: int, total: int, device, check_contiguous: bool = True):
    """Per-row attended slot range [start, end) from an HF decode mask.

    Returns (starts, ends) int32 device tensors, or (None, None) without a mask.  The
    kernel attends to every slot of the range, so a row whose attended slots have a
    hole (right padding followed by generated tokens) cannot take this path: with
    ``check_contiguous`` such masks raise ``_HoleyMask`` (one host sync to find out);
    callers that know the mask's shape pass False.  The result for one mask tensor is
    computed once and reused by the following layers of the same forward; a capture
    computes its own, once on a stream too, which every replay then does from the mask as it is.
    A capture cannot look at the mask: what the step before it found of the same mask is taken
    (replays are to have masks of the same kind), and without such a step the call is refused.
    """
    if attention_mask is None:
        return None, None
    if attention_mask.is_cuda and torch.cuda.is_current_stream_capturing():
        if check_contiguous:
            c = getattr(_tls, "last_range", None)
            if c is None or c[0] is not attention_mask or c[1][0] is None or c[1][:5] != (_version(attention_mask), B, total, True, device):
                raise ValueError(_UNKNOWN_MASK)
            if c[2] is None:
                raise _HoleyMask
        at = attention_mask.device
        key = _version(attention_mask), B, total, device, K._stream_handle(at), K.capture_id(at)
        c = getattr(_tls, "captured_range", None)
        if c is None or c[0] is not attention_mask or c[1] != key or key[0] is None:
            # (held until the next mask: the capture's later allocations leave the result alone)
            c = _tls.captured_range = (attention_mask, key, _compute_range(attention_mask, B, total, device, False))
        return c[2]
    _tls.captured_range = None
    key = (_version(attention_mask), B, total, check_contiguous, device,
           K._stream_handle(attention_mask.device) if attention_mask.is_cuda else 0)
    c = getattr(_tls, "last_range", None)
    if c is not None and c[0] is attention_mask and c[1] == key and key[0] is not None:
        if c[2] is None:
            raise _HoleyMask
        return c[2]
    try:
        result = _compute_range(attention_mask, B, total, device, check_contiguous)
    except _HoleyMask:
        _tls.last_range = (attention_mask, key, None)
        raise
    _tls.last_range = (attention_mask, key, result)
    return result


def _compute_range(attention_mask: torch.Tensor, B: int, total: int, device, check_contiguous: bool):
    m = _attend_mask(attention_mask, B, total)
    idx = torch.arange(m.shape[1], device=m.device, dtype=torch.int32)
    big = torch.iinfo(torch.int32).max
    starts = torch.where(m, idx, torch.full_like(idx, big)).amin(dim=1)
    ends = torch.where(m, idx + 1, torch.zeros_like(idx)).amax(dim=1)
    starts = torch.minimum(starts, ends)
    if check_contiguous and bool(((ends - starts) != m.sum(dim=1, dtype=torch.int32)).any()):
        raise _HoleyMask
    return starts.to(device=device, dtype=torch.int32), ends.to(device=device, dtype=torch.int32)


class _HoleyMask(Exception):
    """A decode mask whose attended slots are not one contiguous range per row."""


def _group_buffers(layer: "PackedMSELayer") -> list[dict]:
    """The store's capacity buffers of each channel group of a split layer."""
    s, sc = layer._store, layer._split
    qjl = sc.use_qjl_keys
    out = []
    for sfx, kg, vg in (("", sc.key_normal, sc.value_normal), ("o", sc.key_outlier, sc.value_outlier)):
        out.append({"key": kg, "value": vg, "k_codes": getattr(s, "kc" + sfx), "k_norms": getattr(s, "kn" + sfx),
                    "k_signs": getattr(s, "ks" + sfx) if qjl else None,
                    "k_rnorms": getattr(s, "kr" + sfx) if qjl else None,
                    "v_codes": getattr(s, "vc" + sfx), "v_norms": getattr(s, "vn" + sfx)})
    return out


def fused_attention(query_states: torch.Tensor, packed_layer: "PackedMSELayer", n_kv_groups: int,
                    attention_mask: torch.Tensor | None = None,
                    choice: "BlockChoice | None" = None, scale: float | None = None) -> torch.Tensor | None:
    """Decode attention of [B, Hq, 1, D] queries over a packed layer -> [B, Hq, 1, D].

    The logit scale is 1/sqrt(D) (reference ``triton_kernels.py:285``) unless ``scale`` is given.  Tokens
    kept dense (``quantize_decode=False``) are merged by log-sum-exp.  Outlier-split
    layers go through the channel-group kernel (where the reference returns None and
    its caller takes the chunked path).  The result has the query's dtype; an fp32
    query gets the kernel's fp32 output (no bf16 rounding).

    Returns None (the reference's "not applicable": the caller takes
    ``chunked_turboquant_attention``) for several query tokens, for GQA groups wider
    than the kernels' 8 query heads per KV head, and for a mask whose attended slots are
    not one contiguous range per row.  The cache layer's ``_tq_mask_contiguous`` (set by
    the generation loop from the prompt mask) spares the host sync of that last check.

    A layer told to (``attend_blocks``), or a ``choice`` given here, attends to chosen blocks of the packed tokens.  Where None is
    returned the caller's other path attends to all of them.
    """
    B, Hq, Sq, D = query_states.shape
    if Sq != 1:
        return None  # the caller takes chunked_turboquant_attention (reference contract)
    store = packed_layer._store
    Hkv = store.kc.shape[1] if store is not None else Hq // max(n_kv_groups, 1)
    if Hq // Hkv > K.MAX_GROUP:
        return None
    n_packed = packed_layer.packed_seq_length()
    n_dense = packed_layer._dense_len
    scale = 1.0 / math.sqrt(D) if scale is None else float(scale)
    known = getattr(packed_layer, "_tq_mask_contiguous", None)
    if attention_mask is not None and known is False:
        return None
    try:
        starts, ends = _valid_range(attention_mask, B, n_packed + n_dense, query_states.device,
                                    check_contiguous=known is None)
    except _HoleyMask:
        return None
    # the kernel sees the packed slots only; ends beyond them (dense tokens) are clamped
    p_ends = ends if ends is None or n_dense == 0 else torch.clamp(ends, max=n_packed)
    f32 = query_states.dtype == torch.float32
    kw = dict(n_tokens=n_packed, seq_starts=starts, seq_lens=p_ends, scale=scale, want_f32=f32 or n_dense > 0,
              want_lse=n_dense > 0)
    if packed_layer._outlier_enabled:
        sc = packed_layer._split
        outs = K.decode_attention_groups(query_states, _group_buffers(packed_layer), key_stack=sc.key_stack,
                                         value_stack=sc.value_stack, qjl_stack=sc.qjl_stack, **kw)
    else:
        c = packed_layer.codecs
        q = query_states
        choice = packed_layer._choice if choice is None else choice
        blocks = None
        if choice is not None:
            q = q if q.dtype in K._QUERY_TYPES else q.float()
            blocks = packed_layer.choose_blocks(q, choice, starts, p_ends)
        attend = K.decode_attention if blocks is None else functools.partial(K.block_attention, blocks=blocks)
        outs = attend(q, k_codes=store.kc, k_norms=store.kn, v_codes=store.vc, v_norms=store.vn, key=c.key, value=c.value,
                      k_signs=store.ks, k_rnorms=store.kr, qjl=c.qjl, **kw)
    if n_dense == 0:
        out = outs[1] if f32 else outs
        return out.to(query_states.dtype).view(B, Hq, 1, D)
    _, o_packed, lse_packed = outs
    dk, dv = packed_layer._dense_buf  # capacity buffers: the first n_dense tokens are attended
    if (_native_rows(query_states, dk, dv) and dk.shape[1] * n_kv_groups == Hq
            and K.DenseAttention.takes(query_states, dk.shape[1])):
        # two launches: the dense tokens' partials, and their merge with the packed part.  The torch
        # operations below take ~22 (at B=4, Hq=32, N=8192 and 203 dense tokens 278 us a call, of
        # which the packed part takes 17)
        q = query_states if query_states.dtype == torch.bfloat16 else query_states.float()
        n = K.DenseAttention.split_count(q, dk.shape[1], n_dense, K.DENSE_SPLITS)
        return K.DenseAttention(q, dk.shape[1], n).add(dk, dv, n_dense, 0, n, scale, starts=starts, ends=ends,
                                                       pos0=n_packed, out=query_states.dtype, prev=o_packed,
                                                       prev_lse=lse_packed)
    # dense decode buffer: exact attention on the few generated tokens, merged by LSE
    dk = packed_layer._dense_keys.float().repeat_interleave(n_kv_groups, dim=1)  # [B, Hq, n, D]
    dv = packed_layer._dense_values.float().repeat_interleave(n_kv_groups, dim=1)
    logits = (query_states.float() @ dk.transpose(-2, -1)).squeeze(2) * scale  # [B, Hq, n]
    if starts is not None:
        pos = torch.arange(n_packed, n_packed + n_dense, device=logits.device)
        ok = (pos[None, :] >= starts[:, None]) & (pos[None, :] < ends[:, None])
        logits = logits.masked_fill(~ok[:, None, :], float("-inf"))
    lse_dense = torch.logsumexp(logits, dim=-1)  # [B, Hq]
    m = torch.maximum(lse_packed, lse_dense)
    m = torch.where(torch.isfinite(m), m, torch.zeros_like(m))
    wp = torch.exp(lse_packed - m)
    wd = torch.exp(logits - m[..., None])  # [B, Hq, n]
    num = o_packed * wp[..., None] + (wd[..., None] * dv).sum(dim=2)
    den = (wp + wd.sum(dim=-1)).clamp(min=1e-30)[..., None]
    return (num / den).to(query_states.dtype).view(B, Hq, 1, D)


_DEFAULT_CHUNK_SIZE = 1024


def triton_available() -> bool:
    """Reference API (runtime/triton_kernels.py): whether the fused decode kernels are usable.
    Here that is libtq.so (there is no Triton in this build)."""
    try:
        _lib.load()
    except (ImportError, OSError):
        return False
    return True


def _repeat_kv(t: torch.Tensor, n_rep: int) -> torch.Tensor:
    return t if n_rep == 1 else t.repeat_interleave(n_rep, dim=1)


def _native_rows(query: torch.Tensor, *rows: torch.Tensor) -> bool:
    """Whether libtq's attention over bf16 rows takes this query and these keys and values.
    Autograd needs torch operations, as do the callers of ``K.torch_operations_watched``; rows of
    another dtype would be rounded."""
    dev, grad = query.device, torch.is_grad_enabled()
    if (dev.type != "cuda" or query.shape[-1] != K.HEAD_DIM or query.dtype == torch.float64 or query.numel() == 0
            or (grad and query.requires_grad) or K.torch_operations_watched()):
        return False
    for t in rows:
        if (t.dtype != torch.bfloat16 or t.device != dev or t.dim() != 4 or t.shape[0] != query.shape[0]
                or t.shape[3] != K.HEAD_DIM or (grad and t.requires_grad) or t.data_ptr() % 16):
            return False
        s0, s1, s2, s3 = t.stride()
        if s3 != 1 or (s0 | s1 | s2) % 8:
            return False
    return True


def _native_mask(mask: torch.Tensor | None, query: torch.Tensor, total: int) -> bool:
    """Whether libtq takes the mask: bool or fp32 (after ``_additive_mask``'s conversion), four
    dimensions that broadcast over [B, Q, Sq] and cover every token."""
    if mask is None:
        return True
    if mask.dim() != 4 or mask.device != query.device or mask.requires_grad or mask.stride(-1) != 1:
        return False
    return (mask.dtype == torch.bool or mask.is_floating_point()) and mask.shape[3] >= total and \
        all(m in (1, n) for m, n in zip(mask.shape[:3], query.shape[:3]))


#: bytes of decoded key and value rows held at once by the native chunked path (at least chunk_size
#: tokens): 64 MiB is 16384 tokens of 8 KV heads, enough to fill the device, and stays in the
#: 256 MB last-level cache between the decoder and the attention
_ROW_BYTES = 64 << 20


def _native_chunked(query: torch.Tensor, layer: "PackedMSELayer", new_key, new_value, mask, chunk_size: int,
                    kv_heads: int, scale: float) -> torch.Tensor:
    """``chunked_turboquant_attention`` in libtq kernels: per segment of the packed history two
    decoder launches and one attention launch, one launch per dense part, one merge of the
    splits."""
    q = query if query.dtype == torch.bfloat16 else query.float()
    if mask is not None and mask.dtype != torch.bool:
        mask = mask.float()
    n_packed = layer.packed_seq_length()
    step = max(int(chunk_size), _ROW_BYTES // (query.shape[0] * kv_heads * K.HEAD_DIM * 4), 1)
    count = lambda n, most: K.DenseAttention.split_count(q, kv_heads, n, most)  # noqa: E731
    ranges = []  # (keys, values, tokens, slots, first slot, continued): keys are None for packed tokens
    slots = 0
    if n_packed:
        slots = count(min(step, n_packed), K.DENSE_SPLITS - 16)
        ranges += [(None, None, min(step, n_packed - a), slots, 0, a > 0) for a in range(0, n_packed, step)]
    for k, v in ((layer._dense_keys, layer._dense_values), (new_key, new_value)):
        if k is not None and k.shape[2]:
            n = count(k.shape[2], 8)
            ranges.append((k, v, k.shape[2], n, slots, False))
            slots += n
    att = K.DenseAttention(q, kv_heads, slots)
    off, out = 0, None
    for i, (k, v, n, splits, first, more) in enumerate(ranges):
        if k is None:
            k, v = layer._key_rows(off, off + n), layer._value_rows(off, off + n)
        out = att.add(k, v, n, first, splits, scale, mask=None if mask is None else mask[..., off:off + n],
                      accumulate=more, out=query.dtype if i + 1 == len(ranges) else None)
        off += n
    return out


def _additive_mask(mask: torch.Tensor | None) -> torch.Tensor | None:
    if mask is None:
        return None
    if mask.dtype == torch.bool:
        return torch.zeros(mask.shape, dtype=torch.float32, device=mask.device).masked_fill(~mask, float("-inf"))
    return mask.float()


def chunked_turboquant_attention(query_states: torch.Tensor, packed_layer: "PackedMSELayer",
                                 new_key: torch.Tensor | None = None, new_value: torch.Tensor | None = None,
                                 n_kv_groups: int = 1, attention_mask: torch.Tensor | None = None,
                                 chunk_size: int = _DEFAULT_CHUNK_SIZE, scale: float | None = None) -> torch.Tensor:
    """Any-shape attention over a packed layer -> [B, Q, Sq, D] (reference runtime/attention.py:215-304).

    The packed history is decoded by libtq ``chunk_size`` tokens at a time into bf16 K / V
    rows (reference ``_decode_keys_range`` / ``_decode_values_range``), then the dense decode
    buffer and ``new_key`` / ``new_value`` follow; logits are fp32 ``q . K / sqrt(D)`` (or times ``scale``) plus
    the mask slice of each part, merged by an online softmax and normalised with the 1e-8
    clamp.  A boolean mask (True = attend) is applied as 0 / -inf; the reference adds
    ``mask.float()``, which is only right for additive masks.  Rows with nothing to attend
    to return zeros (the reference's running maximum turns them into NaN).
    """
    B, Q, Sq, D = query_states.shape
    scale = 1.0 / math.sqrt(D) if scale is None else float(scale)
    dense = (packed_layer._dense_keys, packed_layer._dense_values)
    parts = [t for t in (*dense, new_key, new_value) if t is not None]
    n_packed = packed_layer.packed_seq_length()
    total = n_packed + sum(int(t.shape[2]) for t in (dense[0], new_key) if t is not None)
    if (total and chunk_size > 0 and Q % max(n_kv_groups, 1) == 0 and (new_key is None) == (new_value is None)
            and (n_packed == 0 or packed_layer.dtype in (torch.bfloat16, torch.float32))
            and _native_rows(query_states, *parts) and _native_mask(attention_mask, query_states, total)
            and all(t.shape[1] * n_kv_groups == Q for t in parts)
            and K.DenseAttention.takes(query_states, Q // n_kv_groups)
            and all(a is None or a.shape == b.shape for a, b in ((dense[0], dense[1]), (new_key, new_value)))
            and (n_packed == 0 or packed_layer._shape == (B, Q // n_kv_groups, D))):
        return _native_chunked(query_states, packed_layer, new_key, new_value, attention_mask, chunk_size,
                               Q // n_kv_groups, scale)
    qf = query_states.float()
    mask = _additive_mask(attention_mask)
    m = torch.full((B, Q, Sq, 1), float("-inf"), device=qf.device)
    s = torch.zeros(B, Q, Sq, 1, device=qf.device)
    o = torch.zeros(B, Q, Sq, D, device=qf.device)
    off = 0

    def attend(keys: torch.Tensor, values: torch.Tensor) -> None:
        nonlocal m, s, o, off
        n = int(keys.shape[-2])
        logits = (qf @ _repeat_kv(keys, n_kv_groups).float().transpose(-2, -1)) * scale
        if mask is not None:
            logits = logits + mask[..., off:off + n]
        new_m = torch.maximum(m, logits.amax(dim=-1, keepdim=True))
        safe = torch.where(torch.isfinite(new_m), new_m, torch.zeros_like(new_m))
        corr = torch.exp(m - safe)
        e = torch.exp(logits - safe)
        s = s * corr + e.sum(dim=-1, keepdim=True)
        o = o * corr + e @ _repeat_kv(values, n_kv_groups).float()
        m = new_m
        off += n

    for a in range(0, n_packed, chunk_size):
        b = min(a + chunk_size, n_packed)
        attend(packed_layer._decode_keys_range(a, b), packed_layer._decode_values_range(a, b))
    if packed_layer._dense_keys is not None:
        attend(packed_layer._dense_keys, packed_layer._dense_values)
    if new_key is not None:
        attend(new_key, new_value)
    return (o / s.clamp(min=1e-8)).to(query_states.dtype)


def _tree_mask(parents: torch.Tensor, total: int, starts: torch.Tensor | None, ends: torch.Tensor) -> torch.Tensor:
    """bool [B, 1, T, total]: the slots each node of a tree attends to; ``parents`` [B, T], ``ends`` [B] each
    row's history end, where its nodes begin."""
    T = parents.shape[1]
    i = torch.arange(T, device=parents.device)
    p = torch.where((parents >= 0) & (parents < i), parents, -1).long()
    sees = torch.eye(T, dtype=torch.bool, device=p.device).expand(p.shape[0], T, T).clone()
    for _ in range(max(1, (T - 1).bit_length())):  # paths of 1, 2, 4, ... steps
        at, live = p.clamp(min=0), p >= 0
        sees |= live[..., None] & sees.gather(1, at[..., None].expand_as(sees))
        p = torch.where(live, p.gather(1, at), -1)
    slot = torch.arange(total, device=p.device)[None, :]
    node = slot - ends[:, None]
    mine = (node >= 0) & (node < T)
    seen = sees.gather(2, node.clamp(0, T - 1)[:, None].expand(-1, T, -1)) & mine[:, None]
    history = node < 0
    if starts is not None:
        history = history & (slot >= starts[:, None])
    return (seen | history[:, None])[:, None]


def tree_attention(query_states: torch.Tensor, packed_layer: "PackedMSELayer", parents: torch.Tensor,
                   n_kv_groups: int | None = None, seq_starts: torch.Tensor | None = None,
                   seq_lens: torch.Tensor | None = None) -> torch.Tensor:
    """Attention of a tree of drafted tokens, [B, Hq, T, D] over a packed layer -> [B, Hq, T, D].

    The T drafted tokens are the layer's last ones (``update`` has stored them, packed or dense as the layer keeps
    generated tokens).  ``parents`` int [T] or [B, T]: the node each follows, an earlier one, or -1; a
    node attends to the history, to its ancestors and to itself (a chain -1, 0, 1, ... is causal).
    ``seq_starts`` / ``seq_lens`` int [B]: row b's history is the tokens [start, len) and its nodes the T
    tokens from len on (packed nodes only).  ``n_kv_groups`` (query heads per KV head) follows from the shapes; another
    number is refused.  After the drafts are checked, ``keep_tokens`` of the layer closes
    up the accepted path.

    One-group layers with up to 64 nodes run on the packed codes (``kernels.tree_attention``), tokens kept
    dense merged by log-sum-exp; others take ``chunked_turboquant_attention`` with the tree as its mask.
    """
    B, Hq, T, D = query_states.shape
    if parents.dim() not in (1, 2) or tuple(parents.shape) not in ((T,), (B, T)):
        raise ValueError(f"parents must be [{T}] or [{B}, {T}], got {tuple(parents.shape)}")
    K._no_gradient("tree_attention", query_states)
    n_packed, n_dense = packed_layer.packed_seq_length(), packed_layer._dense_len
    total = n_packed + n_dense
    if T > (n_dense if n_dense else n_packed):
        raise ValueError(f"{T} drafted tokens, but the layer holds {n_dense or n_packed} of their kind")
    if n_dense and seq_lens is not None:
        raise ValueError("seq_lens needs the drafted tokens packed (quantize_decode=True)")
    store = packed_layer._store
    if total == 0:  # no nodes either
        return torch.empty_like(query_states)
    batch, kv_heads = (store.B, store.H) if store is not None else packed_layer._dense_buf[0].shape[:2]
    if batch != B or Hq % kv_heads or n_kv_groups not in (None, Hq // kv_heads):
        raise ValueError(f"queries {tuple(query_states.shape)} with n_kv_groups {n_kv_groups} do not match a layer of "
                         f"{batch} rows and {kv_heads} KV heads")
    n_kv_groups = Hq // kv_heads
    dev = query_states.device
    seq_starts = K._int32_on(seq_starts, dev, "seq_starts", (B,))
    seq_lens = K._int32_on(seq_lens, dev, "seq_lens", (B,))
    fused = (store is not None and not packed_layer._outlier_enabled and T <= K.MAX_NODES
             and query_states.dtype in K._QUERY_TYPES)
    if fused:
        c = packed_layer.codecs
        kw = dict(k_codes=store.kc, k_norms=store.kn, v_codes=store.vc, v_norms=store.vn, n_tokens=n_packed, key=c.key,
                  value=c.value, k_signs=store.ks, k_rnorms=store.kr, qjl=c.qjl, seq_starts=seq_starts)
        if n_dense == 0:
            return K.tree_attention(query_states, parents, seq_lens=seq_lens, **kw)
    own = parents.to(dev)
    own = own[None].expand(B, -1) if own.dim() == 1 else own
    ends = torch.full((B,), total - T, dtype=torch.int32, device=dev) if seq_lens is None else seq_lens
    if fused:
        dk, dv = packed_layer._dense_buf
        if _native_rows(query_states, dk, dv) and K.DenseAttention.takes(query_states, dk.shape[1]):
            _, o_packed, lse = K.tree_attention(query_states, None, want_f32=True, want_lse=True, **kw)
            starts = None if seq_starts is None else seq_starts - n_packed
            mask = _tree_mask(own, n_dense, starts, ends - n_packed)
            q = query_states if query_states.dtype == torch.bfloat16 else query_states.float()
            n = K.DenseAttention.split_count(q, dk.shape[1], n_dense, K.DENSE_SPLITS)
            return K.DenseAttention(q, dk.shape[1], n).add(dk, dv, n_dense, 0, n, 1.0 / math.sqrt(D), mask=mask,
                                                           out=query_states.dtype, prev=o_packed, prev_lse=lse)
    return chunked_turboquant_attention(query_states, packed_layer, n_kv_groups=n_kv_groups,
                                        attention_mask=_tree_mask(own, total, seq_starts, ends))


def block_sparse_attention(query_states: torch.Tensor, packed_layer: "PackedMSELayer", keep: int, sink: int = 1, recent: int = 2,
                           attention_mask: torch.Tensor | None = None) -> torch.Tensor:
    """A decode step [B, Hq, 1, D] over ``keep`` blocks of 64 packed tokens for each KV head -> [B, Hq, 1, D].

    The first ``sink`` blocks, the last ``recent`` and those that the query heads may give the largest logits, by bounds of the
    keys that the layer keeps (``PackedMSELayer.attend_blocks`` has every step of a model do it); tokens kept dense are all attended
    to.  A history of no more blocks is attended to in full.  One-group layers, up to 8 query heads per KV head, masks of one
    range per row; others, which a model's step would attend to in full, are refused."""
    from turboquant.runtime.packed_qmse_cache import BlockChoice

    B, Hq, Sq, D = query_states.shape
    store = packed_layer._store
    if store is None or packed_layer._outlier_enabled or (B, D) != (store.B, K.HEAD_DIM) or Sq != 1 or Hq % store.H \
            or Hq // store.H > K.MAX_GROUP:
        raise ValueError(f"block_sparse_attention takes one query token per row of a packed one-group layer and up to "
                         f"{K.MAX_GROUP} query heads per KV head, got {tuple(query_states.shape)}")
    out = fused_attention(query_states, packed_layer, Hq // store.H, attention_mask, BlockChoice(keep, sink, recent))
    if out is None:
        raise ValueError("block_sparse_attention: a row's attended tokens must be one range")
    return out


def _shared_ranges(layer: "SharedPrefixLayer", mask: torch.Tensor | None, device):
    """(prefix starts, prefix ends, own ends) of a step's mask, int32 or None.

    ``_HoleyMask`` where a row's tokens are not one range, or where the sequences of a prompt do not share its padding: a host
    sync to find out, which a caller spares who knows and says so in the layer's ``_tq_mask_contiguous``: True, every mask is
    of such ranges, or False (as for ``fused_attention``).  In a captured step what the step before found of the mask counts."""
    if mask is None:
        return None, None, None
    known = getattr(layer, "_tq_mask_contiguous", None)
    if known is False:
        raise _HoleyMask
    n = layer.prefix.packed_seq_length()
    starts, ends = _valid_range(mask, layer.batch, layer.get_seq_length(), device, check_contiguous=not known)
    first, last = starts[layer.first_of], ends.clamp(max=n)[layer.first_of]
    if not known:
        key = _version(mask), layer.counts, n, layer.get_seq_length()
        c = getattr(_tls, "last_shared", None)
        seen = c is not None and c[0] is mask and c[1] == key and key[0] is not None
        if mask.is_cuda and torch.cuda.is_current_stream_capturing():
            if not seen:
                raise ValueError(_UNKNOWN_MASK)
            apart = c[2]
        else:
            apart = bool(((starts != first[layer.prompt_of]) | (ends.clamp(max=n) != last[layer.prompt_of]) | (starts > n)).any())
            _tls.last_shared = mask, key, apart
        if apart:
            raise _HoleyMask
    return first, last, (ends - n).clamp(min=0)


def _rows_mask(mask: torch.Tensor | None, B: int, Sq: int, total: int, device) -> torch.Tensor | None:
    """The mask of a batch's last ``Sq`` of ``total`` tokens in four dimensions; without one, and of one [B, total], each sees those up to
    its own."""
    if mask is not None and mask.dim() == 4:
        return mask[..., :total] if mask.dtype == torch.bool or mask.is_floating_point() else mask[..., :total] != 0
    seen = None if mask is None else _attend_mask(mask, B, total)[:, None, None]
    if Sq == 1:
        return seen
    up_to = torch.ones(Sq, total, dtype=torch.bool, device=device).tril(total - Sq)[None, None]
    return up_to if seen is None else up_to & seen


def shared_prefix_attention(query_states: torch.Tensor, layer: "SharedPrefixLayer",
                            attention_mask: torch.Tensor | None = None, scale: float | None = None) -> torch.Tensor:
    """Attention of sequences that continue shared packed prompts, [B, Hq, Sq, D] over a ``SharedPrefixLayer`` -> [B, Hq, Sq, D].

    One query token per sequence, up to 64 query heads per KV head and a mask of one range per row (left padding of the
    prompts) run on the packed codes (``kernels.prefix_attention``), tokens kept dense merged by log-sum-exp; others
    take the decoded rows (``chunked_turboquant_attention``), the Sq tokens being the sequences' last ones.  The logit scale is
    1/sqrt(D) unless ``scale`` is given."""
    B, Hq, Sq, D = query_states.shape
    scale = 1.0 / math.sqrt(D) if scale is None else float(scale)
    prefix, own = layer.prefix, layer.own
    store, n_prefix, n_own, n_dense = prefix._store, prefix.packed_seq_length(), own.packed_seq_length(), own._dense_len
    if B != layer.batch or Hq % store.H:
        raise ValueError(f"queries {tuple(query_states.shape)} for {layer.batch} sequences and {store.H} KV heads")
    group, dev = Hq // store.H, query_states.device
    dense = own._dense_buf if n_dense else ()
    if (Sq == 1 and group <= 64 and query_states.dtype in K._QUERY_TYPES and _native_rows(query_states, *dense)
            and (not n_dense or K.DenseAttention.takes(query_states, store.H))):
        try:
            starts, ends, own_ends = _shared_ranges(layer, attention_mask, dev)
        except _HoleyMask:
            pass
        else:
            arrays = lambda s: {"k_codes": s.kc, "k_norms": s.kn, "k_signs": s.ks, "k_rnorms": s.kr,  # noqa: E731
                                "v_codes": s.vc, "v_norms": s.vn}
            c = prefix.codecs
            kw = dict(n_prefix=n_prefix, n_own=n_own, key=c.key, value=c.value, qjl=c.qjl, cu_rows=layer.cu_rows,
                      max_rows=max(layer.counts), prefix_starts=starts, prefix_lens=ends, own_lens=own_ends, scale=scale)
            mine = arrays(own._store) if n_own else None
            if not n_dense:
                return K.prefix_attention(query_states, arrays(store), mine, **kw).view(B, Hq, 1, D)
            _, o_packed, lse = K.prefix_attention(query_states, arrays(store), mine, want_f32=True, want_lse=True, **kw)
            q = query_states if query_states.dtype == torch.bfloat16 else query_states.float()
            n = K.DenseAttention.split_count(q, store.H, n_dense, K.DENSE_SPLITS)
            more = {} if own_ends is None else dict(starts=torch.zeros_like(own_ends), ends=own_ends, pos0=n_own)
            return K.DenseAttention(q, store.H, n).add(*dense, n_dense, 0, n, scale, out=query_states.dtype,
                                                       prev=o_packed, prev_lse=lse, **more)
    keys, values = layer.dense_rows()
    mask = _rows_mask(attention_mask, B, Sq, keys.shape[2], dev)
    return chunked_turboquant_attention(query_states, layer.without_tokens(), keys, values, group, mask, scale=scale)


def prompt_attention(query: torch.Tensor, key: torch.Tensor, value: torch.Tensor, *,
                     cu_seqlens: torch.Tensor | None = None, seq_starts: torch.Tensor | None = None,
                     seq_ends: torch.Tensor | None = None, scale: float | None = None,
                     out: torch.Tensor | None = None, return_lse: bool = False):
    """Causal attention over whole prompts, [B, Hq, S, D] against [B, Hkv, S, D] (bf16 or fp16) -> [B, Hq, S, D].

    A padded batch gives each row's [``seq_starts``, ``seq_ends``); prompts packed behind one another (B = 1)
    give ``cu_seqlens``.  See ``kernels.prompt_attention``."""
    return K.prompt_attention(query, key, value, cu_seqlens=cu_seqlens, seq_starts=seq_starts, seq_ends=seq_ends,
                              scale=scale, out=out, want_lse=return_lse)


def _sdpa_fallback(module, query, key, value, attention_mask, scaling):
    """Standard SDPA for prefill and norm-guarded dense layers (reference :75-99)."""
    causal = attention_mask is None and query.shape[-2] > 1
    n_kv_groups = getattr(module, "num_key_value_groups", 1)
    out = F.scaled_dot_product_attention(query, key, value, attn_mask=attention_mask, dropout_p=0.0,
                                         is_causal=causal, scale=scaling, enable_gqa=n_kv_groups > 1)
    return out.transpose(1, 2).contiguous(), None


def _hands_over_all(layer: "PackedMSELayer", query: torch.Tensor, key: torch.Tensor,
                    attention_mask: torch.Tensor | None) -> bool:
    """Whether the call's own keys are all that its rows attend to.

    A layer with the backend wired hands over the new tokens alone.  They are everything where it held nothing
    before them: at a first prompt, and at the one after ``crop`` or ``keep_tokens`` left nothing.  Where that prompt
    has been packed, its rows attend to the exact keys, each up to its own token, as those of a prompt that is packed
    afterwards do; a call with a mask has its rows' ranges there, and takes the packed tokens."""
    if layer._force_dense:
        return True
    packed, Sq = layer.packed_seq_length(), query.shape[-2]
    if packed == 0:
        return layer._dense_len <= key.shape[-2]
    return (Sq > 1 and attention_mask is None and Sq == packed + layer._dense_len and key is not None
            and key.shape[-2] == Sq)


def turboquant_attention_forward(module: torch.nn.Module, query: torch.Tensor, key: torch.Tensor,
                                 value: torch.Tensor, attention_mask: torch.Tensor | None, dropout: float = 0.0,
                                 scaling: float | None = None, is_causal: bool | None = None, **kwargs):
    """HF attention-interface function: returns ([B, Sq, Hq, D], None).  Logits are scaled by ``scaling`` (1/sqrt(D) without) on every
    path, the prompt's before a layer is packed and the steps over it alike; the reference's steps leave it out
    (``triton_kernels.py:285``)."""
    layer = getattr(module, "_tq_cache_layer", None)
    if getattr(layer, "shares_prompts", False):
        scale = None if scaling is None else K._logit_scale("shared_prefix_attention", scaling)
        return shared_prefix_attention(query, layer, attention_mask, scale).transpose(1, 2).contiguous(), None
    if layer is None or _hands_over_all(layer, query, key, attention_mask):
        return _sdpa_fallback(module, query, key, value, attention_mask, scaling)
    if layer.packed_seq_length() == 0:  # the tokens before are dense: attended to as a norm-guarded layer's are
        Sq, held = query.shape[-2], layer._dense_len
        if attention_mask is None and Sq > 1:
            attention_mask = torch.ones(Sq, held, dtype=torch.bool, device=query.device).tril(held - Sq)
        return _sdpa_fallback(module, query, layer._dense_keys, layer._dense_values, attention_mask, scaling)
    n_kv_groups = getattr(module, "num_key_value_groups", 1)
    scale = None if scaling is None else K._logit_scale("fused_attention", scaling)
    out = fused_attention(query, layer, n_kv_groups, attention_mask, scale=scale) if query.shape[-2] == 1 else None
    if out is None:  # several query tokens, or a shape / mask the fused kernel does not take
        out = chunked_turboquant_attention(query, layer, n_kv_groups=n_kv_groups, attention_mask=attention_mask, scale=scale)
    return out.transpose(1, 2).contiguous(), None


def _sequences_mask(cu: torch.Tensor, cu_k: torch.Tensor, rows: int, keys: int, causal: bool, window: int | None,
                    device: torch.device) -> torch.Tensor:
    """bool [rows, keys]: the keys each row of sequences packed behind one another attends to; a sequence's rows and keys end
    together."""
    def ranges(offsets: torch.Tensor, n: int):  # each place's sequence, how far from its end, and whether it is of any
        offsets, at = offsets.to(device).long(), torch.arange(n, device=device)
        seq = torch.searchsorted(offsets[1:].contiguous(), at, right=True)
        left = offsets[1:][seq.clamp(max=offsets.numel() - 2)] - at
        return seq, left, (at >= offsets[0]) & (at < offsets[-1])

    (seq, left, live), (seq_k, left_k, live_k) = ranges(cu, rows), ranges(cu_k, keys)
    mask = (seq[:, None] == seq_k[None, :]) & live[:, None] & live_k[None, :]
    back = left_k[None, :] - left[:, None]  # 0: the row's own token
    if causal:
        mask &= back >= 0
    if window is not None:
        mask &= back < window
    return mask


def turboquant_prompt_forward(module: torch.nn.Module, query: torch.Tensor, key: torch.Tensor, value: torch.Tensor,
                              attention_mask: torch.Tensor | None, dropout: float = 0.0,
                              scaling: float | None = None, is_causal: bool | None = None, **kwargs):
    """HF attention-interface function "turboquant_prompt": whole causal prompts without a mask, alone or packed
    (``cu_seq_lens_q``, a batch of 1), go through ``prompt_attention``; what it does not take (a mask, dropout, a gradient, a trace or a
    transform, other types, head sizes and keys than the prompt's own) and layers that hold earlier tokens go the way of "turboquant".
    Packed sequences keep to themselves there too, by a mask made from their offsets; one that is given counts instead of them.
    One tensor as ``cu_seq_lens_q`` and ``cu_seq_lens_k`` spares a host sync that compares them."""
    causal = getattr(module, "is_causal", True) if is_causal is None else is_causal
    window = kwargs.get("sliding_window")
    cu, cu_k = kwargs.get("cu_seq_lens_q"), kwargs.get("cu_seq_lens_k")
    S = query.shape[-2]
    layer = getattr(module, "_tq_cache_layer", None)
    if getattr(layer, "shares_prompts", False):
        if cu is not None and cu.numel() > 2 and attention_mask is None and S > 1:
            raise ValueError("packed sequences, but the cache layer holds tokens before them")
        if not causal and attention_mask is None and S > 1:  # no mask means causal there
            attention_mask = torch.ones(S, layer.get_seq_length(), dtype=torch.bool, device=query.device).expand(query.shape[0], 1, -1, -1)
        return turboquant_attention_forward(module, query, key, value, attention_mask, dropout, scaling, is_causal, **kwargs)
    if (attention_mask is None and causal and not dropout and S > 1 and query.shape[-1] == K.HEAD_DIM
            and key.shape == value.shape and key.shape[-2:] == query.shape[-2:] and query.is_cuda
            and query.dtype in (torch.bfloat16, torch.float16) and key.dtype == value.dtype == query.dtype
            and (window is None or window >= S) and kwargs.get("softcap") is None and kwargs.get("s_aux") is None
            and (cu is None or (query.shape[0] == 1 and (cu_k is None or cu_k is cu or torch.equal(cu_k, cu))))
            and not K.torch_operations_watched()
            and not (torch.is_grad_enabled() and (query.requires_grad or key.requires_grad or value.requires_grad))):
        if layer is None or _hands_over_all(layer, query, key, attention_mask):
            return prompt_attention(query, key, value, cu_seqlens=cu, scale=scaling).transpose(1, 2), None
    if cu is not None and attention_mask is None and S > 1:
        cu_k = cu if cu_k is None else cu_k
        if query.shape[0] != 1:
            raise ValueError(f"cu_seq_lens_q takes sequences packed into a batch of 1, got {query.shape[0]}")
        if cu_k.numel() != cu.numel():
            raise ValueError("cu_seq_lens_q and cu_seq_lens_k must name as many sequences")
        if layer is None or _hands_over_all(layer, query, key, None):
            mask = _sequences_mask(cu, cu_k, S, key.shape[-2], causal, window, query.device)
            empty = ~mask.any(-1, keepdim=True)  # rows of no sequence, or without keys
            out, _ = _sdpa_fallback(module, query, key, value, mask | empty, scaling)
            return out.masked_fill(empty[None, :, None], 0.0), None
        if cu.numel() > 2:
            raise ValueError("packed sequences, but the cache layer holds tokens before them")
    if not causal and attention_mask is None and S > 1:  # no mask means causal there
        held = key.shape[-2] if layer is None or _hands_over_all(layer, query, key, None) else layer.get_seq_length()
        attention_mask = torch.ones(S, held, dtype=torch.bool, device=query.device).expand(query.shape[0], 1, -1, -1)
    return turboquant_attention_forward(module, query, key, value, attention_mask, dropout, scaling, is_causal, **kwargs)


def _register_attention_backend() -> None:
    """Register "turboquant" and "turboquant_prompt" with HF's attention and mask interfaces (idempotent)."""
    try:
        from transformers.modeling_utils import ALL_ATTENTION_FUNCTIONS
    except ImportError:  # pragma: no cover - transformers is a hard dependency of the adapter
        return
    for name, forward in (("turboquant", turboquant_attention_forward), ("turboquant_prompt", turboquant_prompt_forward)):
        if name not in ALL_ATTENTION_FUNCTIONS:
            ALL_ATTENTION_FUNCTIONS.register(name, forward)
    try:
        from transformers.masking_utils import ALL_MASK_ATTENTION_FUNCTIONS

        for name in ("turboquant", "turboquant_prompt"):
            if name not in ALL_MASK_ATTENTION_FUNCTIONS:
                ALL_MASK_ATTENTION_FUNCTIONS.register(name, ALL_MASK_ATTENTION_FUNCTIONS["sdpa"])
    except (ImportError, KeyError):  # pragma: no cover
        pass


_register_attention_backend()
