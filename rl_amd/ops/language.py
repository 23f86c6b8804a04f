"""Operators of language-model reinforcement learning.

* :func:`token_log_probs` — log-probabilities of given tokens under logits
  (differentiable; csrc/token_loss.hip);
* :func:`token_policy_loss` — the clipped token-level policy loss with its KL
  and entropy terms (differentiable; csrc/token_loss.hip);
* :func:`paged_kv_append` — new keys and values into a paged cache, keys and
  queries rotated to their positions on the way (csrc/paged_kv.hip);
* :func:`paged_attention_decode` — attention of one new token per sequence
  over that cache (csrc/paged_kv.hip).

On a HIP device the kernels run, on the current stream, without a host
synchronisation, with workspaces from torch's allocator: calls can be captured
into a graph.  CPU tensors take the elementary torch forms below.
"""
from __future__ import annotations

import math
from typing import NamedTuple, Optional, Tuple

import torch

from . import _C, _require_ext

__all__ = [
    "TokenPolicyLoss",
    "paged_attention_decode",
    "paged_kv_append",
    "rotary_table",
    "token_log_probs",
    "token_policy_loss",
]

_VARIANTS = {"clip": 0, "cispo": 1}
_fw = torch.autograd.forward_ad


def _native(tensor: torch.Tensor, *others: Optional[torch.Tensor]):
    """The extension for a GPU tensor; None on the CPU (and on a GPU without
    it where the eager fallback is allowed), and where one of the tensors carries a
    forward derivative, which the kernels do not compute."""
    if _fw._current_level >= 0 and any(
            t is not None and _fw.unpack_dual(t).tangent is not None for t in (tensor, *others)):
        return None
    return _C if tensor.is_cuda and _require_ext() else None


def _ordinary(*tensors: torch.Tensor) -> bool:
    """Whether all are tensors whose memory a kernel can take: not subclasses,
    not under functorch's transforms, forward derivatives, a tracing compiler, a
    trace or a mode that sees every operation.  What offers an operator in place of
    elementary torch asks this first."""
    if (
        torch.compiler.is_compiling()
        or _fw._current_level >= 0
        or torch.jit.is_tracing()
        or torch._C._len_torch_dispatch_stack()
    ):
        return False
    return all(
        type(t) in (torch.Tensor, torch.nn.Parameter)
        and not torch._C._functorch.is_functorch_wrapped_tensor(t)
        for t in tensors)


# --------------------------------------------------------------------------- #
# token log-probabilities
# --------------------------------------------------------------------------- #
def token_log_probs(
    logits: torch.Tensor,
    tokens: torch.Tensor,
    *,
    temperature: float = 1.0,
    ignore_index: int = -100,
) -> torch.Tensor:
    """``log_softmax(logits / temperature)`` at ``tokens``, without the
    ``[..., vocab]`` log-probabilities.

    Args:
        logits: ``[..., V]`` in float32, bfloat16 or float16; leading dims may
            be strided (a slice of a longer sequence is not copied).
        tokens: ``[...]`` int64 or int32.  ``ignore_index`` marks places that
            do not count: their log-prob is 0, their logits are not read and
            get a gradient of exactly 0.  Any other token outside ``[0, V)``
            gives NaN (nothing is read out of range).
        temperature: positive (1e-30 to 1e30).

    Returns:
        ``[...]`` float32.  Differentiable in ``logits``; the gradient has
        the logits' dtype, and is itself differentiable in elementary operations
        (``create_graph``), which dual tensors take as well for their forward
        derivatives.  A place with an upstream gradient of 0 gets a gradient of
        exactly 0 whatever its logits hold.  A row of nothing but ``-inf`` gives
        NaN.
    """
    c = _native(logits)
    if c is not None:
        return c.token_log_probs(logits, tokens, temperature, ignore_index)
    if _C is not None:
        _C.token_log_probs_check(logits, tokens, temperature)
    gone = tokens == ignore_index
    known = (tokens >= 0) & (tokens < logits.shape[-1])
    at = torch.where(known, tokens, 0).long().unsqueeze(-1)
    # ignored rows are replaced first: a NaN there would come back through the
    # backward pass as 0 * NaN
    x = torch.where(gone.unsqueeze(-1), 0.0, logits.float() / temperature)
    lp = torch.where(known, x.log_softmax(-1).gather(-1, at).squeeze(-1), torch.nan)
    return torch.where(gone, 0.0, lp)


# --------------------------------------------------------------------------- #
# token policy loss
# --------------------------------------------------------------------------- #
class TokenPolicyLoss(NamedTuple):
    """What :func:`token_policy_loss` returns: float32 scalars.  The first
    four and ``ess`` carry a gradient to ``log_probs``, and the forward derivatives
    of dual tensors, in elementary operations."""

    loss_total: torch.Tensor
    loss_objective: torch.Tensor
    loss_kl: torch.Tensor
    loss_entropy: torch.Tensor
    kl: torch.Tensor
    clip_fraction: torch.Tensor
    ess: torch.Tensor


def token_policy_loss(
    log_probs: torch.Tensor,
    old_log_probs: torch.Tensor,
    advantage: torch.Tensor,
    mask: Optional[torch.Tensor] = None,
    ref_log_probs: Optional[torch.Tensor] = None,
    *,
    clip_low: float = 0.2,
    clip_high: float = 0.2,
    variant: str = "clip",
    kl_coeff: float = 0.0,
    entropy_coeff: float = 0.0,
    reduction: str = "mean",
) -> TokenPolicyLoss:
    """Token-level clipped policy loss with a KL penalty to a reference
    model (the objective of ``GRPOLoss``, ``DAPO`` and ``CISPOLoss``).

    With ``r = exp(log_probs - old_log_probs)`` and the mask's weights ``w``:

    * ``"clip"``: ``gain = min(r A, clip(r, 1 - clip_low, 1 + clip_high) A)``;
    * ``"cispo"``: ``gain = clip(r) log(r) A`` with the weight held constant;
    * ``loss_objective = -sum(w gain) / max(1, sum(w))``;
    * ``kl``: the same mean of ``exp(y) - 1 - y``, ``y = ref - log_probs``;
      ``loss_kl = kl_coeff * kl``;
    * ``loss_entropy``: ``entropy_coeff`` times the mean log-prob (the sampled
      entropy's negative);
    * ``loss_total``: their sum; a term whose coefficient is 0 counts as 0,
      infinite or not;
    * ``clip_fraction``: the share of all places, masked ones too, with
      ``|r - 1| > clip_low``; ``ess``: ``sum(r)^2 / sum(r^2) / numel`` over all
      places (as ``GRPOLoss`` reports them).

    Args:
        log_probs, old_log_probs, ref_log_probs: one shape, float32, bfloat16
            or float16, any strides.  Only ``log_probs`` gets a gradient; the
            others must not require one.
        advantage: broadcasts to ``log_probs``.
        mask: bool, integer or float weights of ``log_probs``' shape, taken in
            float32.  A place of weight 0 may hold anything (the losses' gradient
            there is 0), though what it holds still enters ``clip_fraction`` and
            ``ess``.
        reduction: ``"mean"`` as above, or ``"sum"``: the weighted sums, not
            divided.
    """
    if variant not in _VARIANTS:
        raise ValueError(f"token_policy_loss: variant must be one of {sorted(_VARIANTS)}, got {variant!r}")
    if reduction not in ("mean", "sum"):
        raise ValueError(f"token_policy_loss: reduction must be 'mean' or 'sum', got {reduction!r}")
    c = _native(log_probs, old_log_probs, advantage, mask, ref_log_probs)
    if c is not None:
        return TokenPolicyLoss(*c.token_policy_loss(
            log_probs, old_log_probs, advantage, mask, ref_log_probs, _VARIANTS[variant],
            clip_low, clip_high, kl_coeff, entropy_coeff, reduction == "mean"))
    if _C is not None:
        _C.token_policy_loss_check(
            log_probs, old_log_probs, advantage, mask, ref_log_probs,
            clip_low, clip_high, kl_coeff, entropy_coeff)
    lp, old = log_probs.float(), old_log_probs.float()
    w = torch.ones_like(lp) if mask is None else mask.float()
    gone = w == 0
    every = (lp - old).exp()
    # masked places are replaced before anything is computed of them: a NaN
    # there would come back through the backward pass as 0 * NaN
    lp = torch.where(gone, 0.0, lp)
    log_w = torch.where(gone, 0.0, lp - old)
    ratio = log_w.exp()
    adv = torch.where(gone, 0.0, advantage.float())
    bounded = ratio.clamp(1 - clip_low, 1 + clip_high)
    gain = torch.minimum(ratio * adv, bounded * adv) if variant == "clip" else bounded.detach() * log_w * adv
    count = w.sum().clamp(min=1) if reduction == "mean" else 1.0
    objective = -(gain * w).sum() / count
    # a term without weight is left out: 0 with a gradient of 0, whatever it holds
    loss_kl, entropy = (lp.masked_fill(torch.ones_like(gone), 0.0).sum() for _ in range(2))
    kl = torch.zeros_like(objective)
    if ref_log_probs is not None:
        y = torch.where(gone, 0.0, ref_log_probs.float() - lp)
        kl = ((torch.expm1(y) - y) * w).sum() / count
        if kl_coeff != 0:
            loss_kl = kl_coeff * kl
    if entropy_coeff != 0:
        entropy = entropy_coeff * (lp * w).sum() / count
    off = ((every.detach() - 1).abs() > clip_low).float().mean()
    ess = every.sum().square() / every.square().sum().clamp(min=1e-9) / every.numel()
    return TokenPolicyLoss(
        objective + loss_kl + entropy, objective, loss_kl, entropy, kl.detach(), off, ess)


# --------------------------------------------------------------------------- #
# paged key-value cache
# --------------------------------------------------------------------------- #
def rotary_table(
    positions: int, rotary_dim: int, *, base: float = 10000.0, device=None
) -> Tuple[torch.Tensor, torch.Tensor]:
    """Cosines and sines ``[positions, rotary_dim / 2]`` of the rotation by
    ``position * base ** (-2 i / rotary_dim)``: angles in 64 bits (those of far
    positions lose their phase in 32), rounded once to float32."""
    if rotary_dim < 2 or rotary_dim % 2 or positions < 1:
        raise ValueError(
            f"rotary_table: needs positions >= 1 and an even rotary_dim >= 2, got {positions} and {rotary_dim}")
    half = rotary_dim // 2
    freq = float(base) ** (-torch.arange(half, dtype=torch.float64, device=device) / half)
    angle = torch.arange(positions, dtype=torch.float64, device=device)[:, None] * freq
    return angle.cos().float(), angle.sin().float()


def _turn(x, cos, sin, interleaved):
    """``x [B, T, H, D]`` rotated in float32 by ``cos/sin [B, T, R / 2]``."""
    half = cos.shape[-1]
    one = slice(0, 2 * half, 2) if interleaved else slice(0, half)
    two = slice(1, 2 * half, 2) if interleaved else slice(half, 2 * half)
    cos, sin = cos.unsqueeze(2), sin.unsqueeze(2)
    x = x.float()
    y = x.clone()
    y[..., one] = x[..., one] * cos - x[..., two] * sin
    y[..., two] = x[..., two] * cos + x[..., one] * sin
    return y


def paged_kv_append(
    k: torch.Tensor,
    v: torch.Tensor,
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    page_table: torch.Tensor,
    start: torch.Tensor,
    *,
    lengths: Optional[torch.Tensor] = None,
    q: Optional[torch.Tensor] = None,
    rope: Optional[Tuple[torch.Tensor, torch.Tensor]] = None,
    interleaved: bool = False,
) -> Optional[torch.Tensor]:
    """Write new keys and values into a paged cache, in place.

    Token ``t`` of sequence ``b`` goes to position ``p = start[b] + t``: slot
    ``p % page_size`` of page ``page_table[b, p // page_size]``.

    Args:
        k, v: ``[batch, tokens, kv_heads, dim]`` in the cache's dtype, any
            strides (views of a fused projection are not copied).
        k_cache, v_cache: ``[pages, kv_heads, page_size, dim]`` in float32,
            bfloat16 or float16, rows dense and aligned to 16 bytes;
            ``page_size`` a power of two up to 4096, ``dim`` a multiple of 8
            up to 256.
        page_table: ``[batch, columns]`` int32.
        start: ``[batch]`` int32 or int64, the tokens each sequence holds.
        lengths: ``[batch]``; only the first ``lengths[b]`` tokens count, what
            follows is padding and writes nothing.  Default: all.
        q: ``[batch, tokens, heads, dim]`` queries to rotate along with the
            keys; needs ``rope``.
        rope: ``(cos, sin)``, each ``[positions, rotary_dim / 2]`` float32
            (:func:`rotary_table`): the first ``rotary_dim`` dims of keys and
            queries turn, in float32, rounded once to the cache's dtype.
        interleaved: rotate dims ``(2i, 2i + 1)`` instead of
            ``(i, i + rotary_dim / 2)``.

    A token whose position is negative or past the table's columns, or whose
    page id is outside ``[0, pages)``, is not written.  A position past the
    rotation's table gives NaN.  Two tokens of one call must not share a slot, and
    ``k`` and ``v`` must not lie in the caches.

    Returns:
        The rotated queries (dense; zeros where padding), or None without ``q``.
    """
    c = _native(k_cache)
    if c is not None:
        return c.paged_kv_append(
            k, v, k_cache, v_cache, page_table, start, lengths, q, rope, interleaved)
    if _C is not None:
        _C.paged_kv_append_check(k, v, k_cache, v_cache, page_table, start, lengths, q, rope)
    batch, width = k.shape[:2]
    page_size = k_cache.shape[2]
    step = torch.arange(width, device=k.device)
    position = start.long()[:, None] + step
    live = step < (torch.full_like(start, width) if lengths is None else lengths)[:, None]
    if rope is not None:
        inside = (position >= 0) & (position < rope[0].shape[0])
        row = torch.where(inside, position, 0)
        cos, sin = (torch.where(inside[..., None], t[row], torch.nan) for t in rope)
        k = _turn(k, cos, sin, interleaved).to(k.dtype)
        if q is not None:
            q = _turn(q, cos, sin, interleaved).to(q.dtype)
            q = torch.where(live[..., None, None], q, 0)
    column = torch.div(position, page_size, rounding_mode="floor")
    if page_table.shape[1]:
        held = (column >= 0) & (column < page_table.shape[1])
        page = page_table.long().gather(1, torch.where(held, column, 0))
        b, t = (live & held & (page >= 0) & (page < k_cache.shape[0])).nonzero(as_tuple=True)
        page, slot = page[b, t], position[b, t] % page_size
        k_cache[page, :, slot] = k[b, t]
        v_cache[page, :, slot] = v[b, t]
    return q


def paged_attention_decode(
    q: torch.Tensor,
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    page_table: torch.Tensor,
    lengths: torch.Tensor,
    *,
    scale: Optional[float] = None,
) -> torch.Tensor:
    """Attention of one query token per sequence over its cached keys:
    ``softmax(scale * q k^T) v``, the running maximum and sum in float32.

    Args:
        q: ``[batch, heads, dim]`` in the cache's dtype; ``heads`` a multiple
            of ``kv_heads`` (query head ``h`` reads key head
            ``h // (heads / kv_heads)``).
        k_cache, v_cache, page_table: as in :func:`paged_kv_append`.
        lengths: ``[batch]`` int32 or int64, the keys each sequence sees, the
            new token's own among them; at most the table's columns times
            ``page_size`` are looked at.  0 or less: zeros.
        scale: default ``dim ** -0.5``.

    Keys on pages outside ``[0, pages)`` are left out; slots past a sequence's
    length may hold anything.  What counts has to be finite: an infinite value gives
    infinity or NaN.

    Returns:
        ``[batch, heads, dim]`` in ``q``'s dtype.
    """
    c = _native(q)
    if c is not None:
        return c.paged_attention_decode(q, k_cache, v_cache, page_table, lengths, scale)
    if scale is None:
        scale = 1.0 / math.sqrt(max(1, q.shape[-1]))
    if _C is not None:
        _C.paged_attention_check(q, k_cache, v_cache, page_table, lengths, scale)
    batch, heads, dim = q.shape
    kv_heads, page_size = k_cache.shape[1], k_cache.shape[2]
    if not page_table.shape[1]:
        return torch.zeros_like(q)
    page = page_table.long()
    held = (page >= 0) & (page < k_cache.shape[0])
    page = torch.where(held, page, 0)
    keys = k_cache[page].float().transpose(1, 2).flatten(2, 3)
    values = v_cache[page].float().transpose(1, 2).flatten(2, 3)
    seen = torch.arange(keys.shape[2], device=q.device) < lengths[:, None]
    seen &= held.repeat_interleave(page_size, 1)
    query = q.float().unflatten(1, (kv_heads, heads // kv_heads)) * scale
    score = torch.matmul(query, keys.transpose(-1, -2))
    score = score.masked_fill(~seen[:, None, None], -torch.inf)
    top = score.amax(-1, keepdim=True).clamp(min=torch.finfo(torch.float32).min)
    e = (score - top).exp()
    total = e.sum(-1, keepdim=True)
    values = values.masked_fill(~seen[:, None, :, None], 0)
    out = torch.matmul(e, values) / torch.where(total == 0, 1.0, total)
    return out.flatten(1, 2).to(q.dtype)
