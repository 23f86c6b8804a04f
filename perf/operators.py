"""The language-model operators of ``rl_amd.ops``: what is measured of them.

Four operators carry a reinforcement-learning step of a language model:

* ``log_probs`` — log-probabilities of given tokens under rows of logits,
  forward and backward (``ops.token_log_probs``);
* ``policy_loss`` — the clipped token-level policy loss with its KL term,
  forward and backward (``ops.token_policy_loss``);
* ``append`` — new keys and values into a paged cache, with the position
  rotation of keys and queries on the way (``ops.paged_kv_append``);
* ``attend`` — attention of one new token per sequence over that cache
  (``ops.paged_attention_decode``).

``run`` computes them in elementary torch operations where ``own`` is false
and calls ``rl_amd.ops`` where it is true; ``exact`` gives the definitions in
64 bits.
"""
import math

import torch

own = False

DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
IGNORE = -100


# --------------------------------------------------------------------------- #
# cases
# --------------------------------------------------------------------------- #
def listed():
    return [
        # behaviour log-probs of the tokens one decode step just sampled
        dict(name="log_probs_step", op="log_probs", batch=64, width=1, vocab=50257,
             dtype="bfloat16", temperature=1.0, lo=1, hi=1, strided=False, grad=False),
        # a small model's odd vocabulary in fp32, sampled at a temperature
        dict(name="log_probs_odd", op="log_probs", batch=7, width=37, vocab=503,
             dtype="float32", temperature=0.7, lo=5, hi=37, strided=False, grad=True),
        # an ordinary learning micro-batch, responses padded to the longest
        dict(name="log_probs_learn", op="log_probs", batch=16, width=128, vocab=50257,
             dtype="bfloat16", temperature=1.0, lo=32, hi=128, strided=False, grad=True),
        # a whole rollout batch: the response's rows inside the full logits
        dict(name="log_probs_batch", op="log_probs", batch=256, width=32, vocab=50257,
             dtype="bfloat16", temperature=1.0, lo=32, hi=32, strided=True, grad=True),
        # a small group of short answers, no reference model
        dict(name="policy_loss_step", op="policy_loss", batch=8, width=45, dtype="float32",
             variant="clip", high=0.2, kl=0.0, entropy=0.0, lo=9, hi=45),
        # one rollout batch of the RLHF benchmark, KL to the reference model
        dict(name="policy_loss_rlhf", op="policy_loss", batch=256, width=32, dtype="float32",
             variant="clip", high=0.2, kl=0.05, entropy=0.0, lo=32, hi=32),
        # long reasoning answers of many groups, asymmetric clip, all terms
        dict(name="policy_loss_long", op="policy_loss", batch=1024, width=4096, dtype="float32",
             variant="clip", high=0.28, kl=0.05, entropy=0.01, lo=200, hi=4096),
        # the cache write of one decode step (learned positions: no rotation)
        dict(name="append_step", op="append", batch=256, width=1, heads=12, kv_heads=12, dim=64,
             dtype="bfloat16", page=16, rotary=0, interleaved=False, lo=1, hi=1, past=96),
        # a batch of ragged prompts, keys and queries rotated
        dict(name="append_prompt", op="append", batch=16, width=2048, heads=32, kv_heads=8, dim=128,
             dtype="bfloat16", page=64, rotary=128, interleaved=False, lo=500, hi=2048, past=0),
        # one decode step of the RLHF benchmark's rollout
        dict(name="attend_step", op="attend", batch=256, heads=12, kv_heads=12, dim=64,
             dtype="bfloat16", page=16, lo=65, hi=96),
        # a ragged serving batch with shared key heads
        dict(name="attend_ragged", op="attend", batch=48, heads=32, kv_heads=8, dim=128,
             dtype="float16", page=64, lo=1, hi=8192),
        # one very long conversation: the split over the cache carries it
        dict(name="attend_long", op="attend", batch=1, heads=32, kv_heads=8, dim=128,
             dtype="bfloat16", page=64, lo=131072, hi=131072),
    ]


def _size(rng, lo, hi):
    """A whole number in [lo, hi], spread over its logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["log_probs", "policy_loss", "append", "attend"])
    if op == "log_probs":
        dtype = rng.choice(["bfloat16", "bfloat16", "float16", "float32"])
        vocab = _size(rng, 200, 160000)
        most = 8192 * 50257 // (2 if dtype == "float32" else 1)
        rows = _size(rng, 1, max(1, min(8192, most // vocab)))
        width = _size(rng, 1, rows)
        grad = rng.random() < 0.75
        return dict(op=op, batch=max(1, rows // width), width=width, vocab=vocab, dtype=dtype,
                    temperature=rng.choice([1.0, 1.0, 0.7, 1.3]),
                    lo=rng.randint(0, width), hi=width, strided=rng.random() < 0.4, grad=grad)
    if op == "policy_loss":
        width = _size(rng, 1, 4096)
        kl = rng.choice([0.0, 0.05, 0.001])
        return dict(op=op, batch=_size(rng, 1, 1024), width=width,
                    dtype=rng.choice(["float32", "float32", "float32", "bfloat16"]),
                    variant=rng.choice(["clip", "clip", "cispo"]), high=rng.choice([0.2, 0.28]),
                    kl=kl, entropy=rng.choice([0.0, 0.01]), lo=rng.randint(0, width), hi=width)
    kv_heads = rng.choice([1, 2, 4, 5, 8, 12])
    heads = kv_heads * rng.choice([1, 1, 2, 3, 4, 7, 8, 16])
    dim = rng.choice([64, 64, 80, 96, 128, 128, 256])
    dtype = rng.choice(["bfloat16", "bfloat16", "float16", "float32"])
    page = rng.choice([8, 16, 32, 64, 128])
    if op == "append":
        most = 16 * 2048 * 48 * 128 // ((heads + 2 * kv_heads) * dim)
        tokens = _size(rng, 1, min(most // 2, 32768))
        width = _size(rng, 1, min(tokens, 4096)) if rng.random() < 0.6 else 1
        return dict(op=op, batch=max(1, min(512, tokens // width)), width=width, heads=heads,
                    kv_heads=kv_heads, dim=dim, dtype=dtype, page=page,
                    rotary=rng.choice([0, dim, dim, dim // 2]), interleaved=rng.random() < 0.4,
                    lo=rng.randint(1, width), hi=width, past=_size(rng, 1, 200))
    most = 48 * 8192 * 8 * 128 // (kv_heads * dim) // (2 if dtype == "float32" else 1)
    most = min(most, 48 * 8192 * 16 // heads)
    hi = _size(rng, 1, min(65536, most))
    batch = _size(rng, 1, max(1, min(256, most // hi)))
    return dict(op=op, batch=batch, heads=heads, kv_heads=kv_heads, dim=dim, dtype=dtype, page=page,
                lo=hi if batch == 1 else rng.randint(0, hi), hi=hi)


def _spread(count, lo, hi):
    """``count`` whole numbers spread evenly over [lo, hi], ``hi`` among them."""
    if count == 1:
        return [hi]
    return [lo + (hi - lo) * i // (count - 1) for i in range(count)]


# --------------------------------------------------------------------------- #
# inputs
# --------------------------------------------------------------------------- #
def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev)
    gen.manual_seed(seed)

    def normal(*shape, std=1.0, dtype=torch.float32):
        return torch.empty(shape, device=dev, dtype=dtype).normal_(0.0, std, generator=gen)

    def order(n):
        return torch.randperm(n, generator=gen, device=dev)

    dtype = DTYPES[case["dtype"]]
    batch = case["batch"]
    lengths = torch.tensor(_spread(batch, case["lo"], case["hi"]), device=dev)[order(batch)]
    s = dict(case=case)
    if case["op"] == "log_probs":
        width, vocab = case["width"], case["vocab"]
        if case["strided"]:
            # prompt and response together; the rows that predict the response
            every = normal(batch, 2 * width + 1, vocab, std=3.0, dtype=dtype)
            logits = every[:, width:2 * width]
        else:
            logits = normal(batch, width, vocab, std=3.0, dtype=dtype)
        tokens = torch.randint(0, vocab, (batch, width), generator=gen, device=dev)
        tokens = torch.where(torch.arange(width, device=dev) < lengths[:, None], tokens, IGNORE)
        s["logits"], s["tokens"] = logits.detach(), tokens
        if case["grad"]:
            s["logits"].requires_grad_()
            s["upstream"] = normal(batch, width)
    elif case["op"] == "policy_loss":
        width = case["width"]
        old = -normal(batch, width).abs() * 2.0
        s["log_probs"] = (old + normal(batch, width, std=0.2)).to(dtype).requires_grad_()
        s["ref"] = (old + normal(batch, width, std=0.3)).to(dtype) if case["kl"] else None
        s["old"] = old.to(dtype)
        s["advantage"] = normal(batch, 1)
        s["mask"] = torch.arange(width, device=dev) < lengths[:, None]
    else:
        heads, kv_heads, dim, page = case["heads"], case["kv_heads"], case["dim"], case["page"]
        width = case.get("width", 1)
        if case["op"] == "append":
            start = torch.tensor(_spread(batch, 0, case["past"]), device=dev)[order(batch)]
            most = case["past"] + width
        else:
            most = case["hi"]
        per = max(1, -(-most // page))
        pages = batch * per + 3
        s["k_cache"] = normal(pages, kv_heads, page, dim, dtype=dtype)
        s["v_cache"] = normal(pages, kv_heads, page, dim, dtype=dtype)
        s["page_table"] = order(pages)[:batch * per].reshape(batch, per).to(torch.int32)
        s["lengths"] = lengths.to(torch.int32)
        if case["op"] == "append":
            # queries, keys and values side by side, as a fused projection leaves them
            rows = normal(batch, width, (heads + 2 * kv_heads) * dim, dtype=dtype)
            q, k, v = rows.split([heads * dim, kv_heads * dim, kv_heads * dim], -1)
            s["q"] = q.unflatten(-1, (heads, dim)) if case["rotary"] else None
            s["k"] = k.unflatten(-1, (kv_heads, dim))
            s["v"] = v.unflatten(-1, (kv_heads, dim))
            s["start"] = start.to(torch.int32)
            if width == 1:
                s["lengths"] = None
            s["rope"] = None
            if case["rotary"]:
                half = case["rotary"] // 2
                freq = 10000.0 ** (-torch.arange(half, device=dev, dtype=torch.float64) / half)
                angle = torch.arange(most, device=dev, dtype=torch.float64)[:, None] * freq
                s["rope"] = (angle.cos().float(), angle.sin().float())
        else:
            s["q"] = normal(batch, heads, dim, dtype=dtype)
    return s


# --------------------------------------------------------------------------- #
# the operators
# --------------------------------------------------------------------------- #
def run(s):
    case = s["case"]
    if own:
        return _OWN[case["op"]](s, case)
    with torch.no_grad():
        return _PLAIN[case["op"]](s, case)


def _own_log_probs(s, case):
    from rl_amd import ops

    if not case["grad"]:
        return {"log_probs": ops.token_log_probs(
            s["logits"], s["tokens"], temperature=case["temperature"], ignore_index=IGNORE)}
    lp = ops.token_log_probs(
        s["logits"], s["tokens"], temperature=case["temperature"], ignore_index=IGNORE)
    (grad,) = torch.autograd.grad(lp, s["logits"], s["upstream"])
    return {"log_probs": lp, "grad": grad}


def _own_policy_loss(s, case):
    from rl_amd import ops

    out = ops.token_policy_loss(
        s["log_probs"], s["old"], s["advantage"], s["mask"], s["ref"],
        clip_low=0.2, clip_high=case["high"], variant=case["variant"],
        kl_coeff=case["kl"], entropy_coeff=case["entropy"])
    (grad,) = torch.autograd.grad(out.loss_total, s["log_probs"])
    return {"loss_total": out.loss_total, "loss_objective": out.loss_objective, "kl": out.kl,
            "loss_entropy": out.loss_entropy, "clip_fraction": out.clip_fraction,
            "ess": out.ess, "grad": grad}


def _own_append(s, case):
    from rl_amd import ops

    q = ops.paged_kv_append(
        s["k"], s["v"], s["k_cache"], s["v_cache"], s["page_table"], s["start"],
        lengths=s["lengths"], q=s["q"], rope=s["rope"], interleaved=case["interleaved"])
    return {"k_cache": s["k_cache"], "v_cache": s["v_cache"], "q": q}


def _own_attend(s, case):
    from rl_amd import ops

    return {"out": ops.paged_attention_decode(
        s["q"], s["k_cache"], s["v_cache"], s["page_table"], s["lengths"])}


def _plain_log_probs(s, case):
    logits, tokens = s["logits"], s["tokens"]
    scale = 1.0 / case["temperature"]
    valid = tokens != IGNORE
    x = logits.float() * scale
    x = x - x.amax(-1, keepdim=True)
    at = torch.where(valid, tokens, 0).unsqueeze(-1)
    picked = x.gather(-1, at).squeeze(-1)
    e = x.exp_()
    total = e.sum(-1)
    out = {"log_probs": torch.where(valid, picked - total.log(), 0.0)}
    if case["grad"]:
        g = torch.where(valid, s["upstream"] * scale, 0.0).unsqueeze(-1)
        d = e.mul_(-g / total.unsqueeze(-1))
        out["grad"] = d.scatter_add_(-1, at, g).to(logits.dtype)
    return out


def _plain_policy_loss(s, case):
    lp, adv, w = s["log_probs"].float(), s["advantage"], s["mask"].float()
    low, high = 0.2, case["high"]
    # 64 bits next to a border of the clip and where exp(x) - 1 - x cancels
    log_w = s["log_probs"].double() - s["old"].double()
    above, below = log_w > math.log1p(high), log_w < math.log1p(-low)
    off = (log_w > math.log1p(low)) | below
    log_w = log_w.float()
    ratio = log_w.exp()
    clipped = torch.where(above, 1 + high, torch.where(below, 1 - low, ratio))
    count = w.sum().clamp(min=1)
    if case["variant"] == "clip":
        # the smaller of both products: the clipped one where it clips against the advantage
        stop = (above & (adv > 0)) | (below & (adv < 0))
        gain = torch.where(stop, clipped, ratio) * adv
        dgain = torch.where(stop, 0.0, ratio * adv)
    else:
        gain = clipped * log_w * adv
        dgain = clipped * adv
    objective = -(gain * w).sum() / count
    grad = case["entropy"] - dgain
    kl = torch.zeros_like(objective)
    if s["ref"] is not None:
        lr = s["ref"].double() - s["log_probs"].double()
        e = lr.expm1()
        kl = ((e - lr).float() * w).sum() / count
        grad = grad - case["kl"] * e.float()
    entropy = case["entropy"] * (lp * w).sum() / count
    return {"loss_total": objective + case["kl"] * kl + entropy, "loss_objective": objective,
            "kl": kl, "loss_entropy": entropy, "clip_fraction": off.float().mean(),
            "ess": ratio.sum().square() / ratio.square().sum().clamp(min=1e-9) / ratio.numel(),
            "grad": (grad * w / count).to(s["log_probs"].dtype)}


def _rotate(x, cos, sin, interleaved):
    """Rotate the first dims of ``x [B, T, H, D]`` in fp32 by ``cos/sin [B, T, R/2]``."""
    half = cos.shape[-1]
    cos, sin = cos.unsqueeze(2), sin.unsqueeze(2)
    x = x.float()
    y = x.clone()
    if interleaved:
        a, b = x[..., 0:2 * half:2], x[..., 1:2 * half:2]
        y[..., 0:2 * half:2] = a * cos - b * sin
        y[..., 1:2 * half:2] = b * cos + a * sin
    else:
        a, b = x[..., :half], x[..., half:2 * half]
        y[..., :half] = a * cos - b * sin
        y[..., half:2 * half] = b * cos + a * sin
    return y


def _plain_append(s, case):
    k, v, q, page = s["k"], s["v"], s["q"], case["page"]
    width = k.shape[1]
    step = torch.arange(width, device=k.device)
    valid = None
    position = s["start"].long()[:, None] + step
    if s["rope"] is not None:
        cos, sin = s["rope"][0][position], s["rope"][1][position]
        q = _rotate(q, cos, sin, case["interleaved"]).to(q.dtype)
        k = _rotate(k, cos, sin, case["interleaved"]).to(k.dtype)
    if s["lengths"] is not None:
        # the padding's places take the last token once more
        valid = step < s["lengths"][:, None]
        source = torch.minimum(step, s["lengths"].long()[:, None] - 1)
        row = torch.arange(k.shape[0], device=k.device)[:, None]
        k, v, position = k[row, source], v[row, source], position.gather(1, source)
        if q is not None:
            q = torch.where(valid[:, :, None, None], q, 0)
    at = s["page_table"].long().gather(1, position // page)
    s["k_cache"].transpose(1, 2)[at, position % page] = k
    s["v_cache"].transpose(1, 2)[at, position % page] = v
    return {"k_cache": s["k_cache"], "v_cache": s["v_cache"], "q": q}


def _plain_attend(s, case):
    q, table = s["q"], s["page_table"].long()
    batch, heads, dim = q.shape
    kv_heads = case["kv_heads"]
    keys = s["k_cache"][table].float().transpose(1, 2).reshape(batch, kv_heads, -1, dim)
    values = s["v_cache"][table].float().transpose(1, 2).reshape(batch, kv_heads, -1, dim)
    seen = (torch.arange(keys.shape[2], device=q.device) < s["lengths"][:, None])[:, None, None]
    query = q.float().reshape(batch, kv_heads, heads // kv_heads, dim) / math.sqrt(dim)
    score = torch.matmul(query, keys.transpose(-1, -2))
    score = torch.where(seen, score, -torch.inf)
    top = score.amax(-1, keepdim=True).clamp(min=torch.finfo(torch.float32).min)
    e = (score - top).exp()
    total = e.sum(-1, keepdim=True)
    out = torch.matmul(e, values) / torch.where(total > 0, total, 1.0)
    return {"out": out.reshape(batch, heads, dim).to(q.dtype)}


_OWN = {"log_probs": _own_log_probs, "policy_loss": _own_policy_loss,
        "append": _own_append, "attend": _own_attend}
_PLAIN = {"log_probs": _plain_log_probs, "policy_loss": _plain_policy_loss,
          "append": _plain_append, "attend": _plain_attend}


# --------------------------------------------------------------------------- #
# what a pass cannot do without
# --------------------------------------------------------------------------- #
def work(case):
    size = 4 if case["dtype"] == "float32" else 2
    counts = _spread(case["batch"], case["lo"], case["hi"])
    if case["op"] == "log_probs":
        read = sum(counts) * case["vocab"]
        every = case["batch"] * case["width"] * case["vocab"]
        if not case["grad"]:
            return {"bytes": read * size, "flops": 3 * read}
        return {"bytes": (read + every) * size, "flops": 7 * read}
    if case["op"] == "policy_loss":
        n = case["batch"] * case["width"]
        arrays = 3 if case["kl"] else 2
        return {"bytes": n * (arrays * size + 1 + size), "flops": 20 * n}
    row = case["dim"] * size
    if case["op"] == "append":
        tokens = sum(counts)
        pads = case["batch"] * case["width"] - tokens
        q = (2 * tokens + pads) * case["heads"] if case["rotary"] else 0
        table = 4 * case["rotary"] * (case["past"] + case["width"])
        return {"bytes": (4 * tokens * case["kv_heads"] + q) * row + table,
                "flops": 3 * tokens * (case["heads"] + case["kv_heads"]) * case["rotary"]}
    keys = sum(counts)
    return {"bytes": (2 * keys * case["kv_heads"] + 2 * case["batch"] * case["heads"]) * row,
            "flops": 4 * keys * case["heads"] * case["dim"]}


# --------------------------------------------------------------------------- #
# the definitions in 64 bits, row by row
# --------------------------------------------------------------------------- #
def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        return _EXACT[case["op"]](s, case)


def _exact_log_probs(s, case):
    logits, tokens = s["logits"].detach(), s["tokens"]
    lp = torch.zeros(tokens.shape, dtype=torch.float64, device=tokens.device)
    grad = None
    if case["grad"]:
        grad = torch.zeros(logits.shape, dtype=torch.float64, device=tokens.device)
    for b in range(tokens.shape[0]):
        keep = (tokens[b] != IGNORE).nonzero().squeeze(-1)
        if not len(keep):
            continue
        z = logits[b][keep].double() / case["temperature"]
        log_p = z - torch.logsumexp(z, -1, keepdim=True)
        here = torch.arange(len(keep), device=tokens.device)
        lp[b, keep] = log_p[here, tokens[b][keep]]
        if case["grad"]:
            d = -log_p.exp()
            d[here, tokens[b][keep]] += 1.0
            grad[b, keep] = d * (s["upstream"][b][keep].double() / case["temperature"]).unsqueeze(-1)
    out = {"log_probs": lp}
    if case["grad"]:
        out["grad"] = grad
    return out


def _exact_policy_loss(s, case):
    lp = s["log_probs"].detach().double().requires_grad_()
    keep = s["mask"]
    count = max(1, int(keep.sum()))
    ratio = torch.exp(lp - s["old"].double())
    adv = s["advantage"].double().expand_as(lp)
    with torch.enable_grad():
        log_w = lp - s["old"].double()
        if case["variant"] == "clip":
            gain = torch.minimum(log_w.exp() * adv, log_w.exp().clamp(0.8, 1 + case["high"]) * adv)
        else:
            gain = log_w.exp().detach().clamp(0.8, 1 + case["high"]) * log_w * adv
        objective = -gain[keep].sum() / count
        kl = torch.zeros((), dtype=torch.float64, device=lp.device)
        if s["ref"] is not None:
            lr = s["ref"].double() - lp
            kl = (torch.expm1(lr) - lr)[keep].sum() / count
        entropy = case["entropy"] * lp[keep].sum() / count
        total = objective + case["kl"] * kl + entropy
        (grad,) = torch.autograd.grad(total, lp)
    n = ratio.numel()
    return {"loss_total": total.detach(), "loss_objective": objective.detach(), "kl": kl.detach(),
            "loss_entropy": entropy.detach(),
            "clip_fraction": (torch.abs(ratio.detach() - 1) > 0.2).double().sum() / n,
            "ess": ratio.detach().sum() ** 2 / (ratio.detach() ** 2).sum() / n, "grad": grad}


def _exact_append(s, case):
    def turned(x):
        x = x.double()
        if s["rope"] is None:
            return x
        y = x.clone()
        for b in range(x.shape[0]):
            first = int(s["start"][b])
            cos, sin = (t[first:first + x.shape[1]].double() for t in s["rope"])
            half = cos.shape[-1]
            if case["interleaved"]:
                one, two = slice(0, 2 * half, 2), slice(1, 2 * half, 2)
            else:
                one, two = slice(0, half), slice(half, 2 * half)
            z = torch.complex(x[b, ..., one], x[b, ..., two]) * torch.complex(cos, sin).unsqueeze(1)
            y[b, ..., one], y[b, ..., two] = z.real, z.imag
        return y

    k, v = turned(s["k"]), s["v"].double()
    q = None if s["q"] is None else turned(s["q"])
    k_cache, v_cache = s["k_cache"].double(), s["v_cache"].double()
    page = case["page"]
    start = s["start"].tolist()
    lengths = [k.shape[1]] * k.shape[0] if s["lengths"] is None else s["lengths"].tolist()
    for b in range(k.shape[0]):
        place = torch.arange(start[b], start[b] + lengths[b], device=k.device)
        at = s["page_table"][b].long()[torch.div(place, page, rounding_mode="floor")]
        k_cache[at, :, place % page] = k[b, :lengths[b]]
        v_cache[at, :, place % page] = v[b, :lengths[b]]
        if q is not None:
            q[b, lengths[b]:] = 0.0
    return {"k_cache": k_cache, "v_cache": v_cache, "q": q}


def _exact_attend(s, case):
    q = s["q"].double()
    out = torch.zeros_like(q)
    group = case["heads"] // case["kv_heads"]
    for b, n in enumerate(s["lengths"].tolist()):
        if not n:
            continue
        at = s["page_table"][b].long()[: -(-n // case["page"])]
        for h in range(case["kv_heads"]):
            k = s["k_cache"][at, h].reshape(-1, case["dim"])[:n].double()
            v = s["v_cache"][at, h].reshape(-1, case["dim"])[:n].double()
            mine = q[b, h * group:(h + 1) * group]
            p = torch.softmax((k @ mine.T) / math.sqrt(case["dim"]), 0)
            out[b, h * group:(h + 1) * group] = (v.T @ p).T
    return {"out": out}


_EXACT = {"log_probs": _exact_log_probs, "policy_loss": _exact_policy_loss,
          "append": _exact_append, "attend": _exact_attend}
