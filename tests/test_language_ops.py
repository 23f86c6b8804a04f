"""The language-model operators against plain 64-bit forms.

``u = 2**-24`` is half a step of float32; an output rounded to ``dtype`` is off
by at most ``finfo(dtype).eps / 2`` of its value (plus half a subnormal step).
"""
import math

import pytest
import torch

from rl_amd import ops

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]
DTYPES = [torch.float32, torch.bfloat16, torch.float16]
U = 2.0 ** -24


def gen(seed):
    g = torch.Generator()
    g.manual_seed(seed)
    return g


def half_step(ref, dtype):
    info = torch.finfo(dtype)
    return ref.abs() * info.eps / 2 + info.tiny * info.eps / 2


def close(got, ref, tol):
    got = got.detach().cpu().double()
    assert got.shape == ref.shape
    assert torch.equal(got.isnan(), ref.isnan())
    ok = ref.isnan() | (got == ref) | ((got - ref).abs() <= tol)
    assert ok.all(), ((got - ref).abs() - tol)[~ok].max()


# --------------------------------------------------------------------------- #
# token_log_probs
# --------------------------------------------------------------------------- #
def log_probs_oracle(logits, tokens, temperature, ignore, upstream):
    z = logits.detach().cpu().double() / temperature
    tokens = tokens.cpu().long()
    live = tokens != ignore
    p = torch.softmax(z, -1)
    at = torch.where(live, tokens, 0).unsqueeze(-1)
    lp = torch.where(live, torch.log_softmax(z, -1).gather(-1, at).squeeze(-1), 0.0)
    g = torch.where(live, upstream.cpu().double() / temperature, 0.0).unsqueeze(-1)
    grad = torch.where(g == 0, 0.0, -g * p)
    grad.scatter_add_(-1, at, g)
    return lp, grad, g, p, z


def log_probs_tolerance(z, g, p, grad, vocab, dtype):
    """Relative error of one exp: its argument (z - m) / T * log2(e) is rounded
    three times, which the exponential turns into 3 u |z - m| / T, and the
    instruction adds 2 u.  Terms far below the maximum weigh nothing, so
    |z - m| / T <= 40 is what counts.  A thread adds at most vocab / 64 terms
    in a row, each rounded.  log and the last sum round the result itself."""
    far = (z.amax(-1, keepdim=True) - z).clamp(max=40).amax(-1, keepdim=True)
    rel = U * (6 * far + vocab / 64 + 32)
    size = (z.amax(-1) - z.amin(-1)).clamp(max=1e30) + math.log(vocab)
    lp_tol = rel.squeeze(-1) + 8 * U * size
    grad_tol = half_step(grad, dtype) * 1.01 + g.abs() * (p * rel + 4 * U * (p + grad.abs() / g.abs().clamp(min=1e-30)))
    return lp_tol, grad_tol


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", [(1, 1), (3, 2), (5, 7), (4, 8), (2, 503), (3, 4097), (2, 50257), (1030, 2049),
                                   (1, 130001), (60, 100003), (65, 100003)])
@pytest.mark.parametrize("temperature", [1.0, 0.7])
def test_log_probs_and_gradient(device, dtype, shape, temperature):
    rows, vocab = shape
    g = gen(rows + vocab)
    logits = (torch.randn(rows, vocab, generator=g) * 4).to(dtype).to(device).requires_grad_()
    tokens = torch.randint(0, vocab, (rows,), generator=g)
    if rows > 2:
        tokens[1] = -100
    tokens = tokens.to(device)
    upstream = torch.randn(rows, generator=g).to(device)
    lp = ops.token_log_probs(logits, tokens, temperature=temperature)
    assert lp.dtype == torch.float32
    (grad,) = torch.autograd.grad(lp, logits, upstream)
    assert grad.dtype == dtype
    want, dwant, gg, p, z = log_probs_oracle(logits, tokens, temperature, -100, upstream)
    lp_tol, grad_tol = log_probs_tolerance(z, gg, p, dwant, vocab, dtype)
    close(lp, want, lp_tol)
    close(grad, dwant, grad_tol)
    with torch.no_grad():
        assert torch.equal(ops.token_log_probs(logits, tokens, temperature=temperature), lp)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_log_probs_large_gradient(dtype):
    """A gradient beyond 128 MB is written past the caches; some of its rows."""
    rows, vocab = 1400, 50257
    g = torch.Generator(device="cuda").manual_seed(0)
    logits = torch.randn(rows, vocab, generator=g, device="cuda").mul_(3).to(dtype).requires_grad_()
    tokens = torch.randint(0, vocab, (rows,), generator=g, device="cuda")
    tokens[5] = -100
    upstream = torch.randn(rows, generator=g, device="cuda")
    lp = ops.token_log_probs(logits, tokens)
    (grad,) = torch.autograd.grad(lp, logits, upstream)
    some = [0, 1, 5, 699, 1398, 1399]
    want, dwant, gg, p, z = log_probs_oracle(logits[some], tokens[some], 1.0, -100, upstream[some])
    lp_tol, grad_tol = log_probs_tolerance(z, gg, p, dwant, vocab, dtype)
    close(lp[some], want, lp_tol)
    close(grad[some], dwant, grad_tol)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", DTYPES)
def test_log_probs_strided_rows(device, dtype):
    """The rows that predict a response, inside the logits of the whole
    sequence; int32 tokens; four leading dims; a transposed layout."""
    g = gen(3)
    whole = torch.randn(3, 9, 131, generator=g).to(dtype).to(device).requires_grad_()
    tokens = torch.randint(0, 131, (3, 4), generator=g).to(device)
    upstream = torch.randn(3, 4, generator=g).to(device)
    lp = ops.token_log_probs(whole[:, 4:8], tokens.int())
    (grad,) = torch.autograd.grad(lp, whole, upstream)
    want, dwant, gg, p, z = log_probs_oracle(whole[:, 4:8], tokens, 1.0, -100, upstream)
    lp_tol, grad_tol = log_probs_tolerance(z, gg, p, dwant, 131, dtype)
    close(lp, want, lp_tol)
    close(grad[:, 4:8], dwant, grad_tol)
    assert (grad[:, :4] == 0).all() and (grad[:, 8:] == 0).all()
    turned = whole[:, 4:8].detach().transpose(1, 2).contiguous().transpose(1, 2)
    assert turned.stride(-1) != 1
    close(ops.token_log_probs(turned, tokens), want, lp_tol)
    many = whole[:, 4:8].detach().reshape(3, 2, 2, 131)[None]
    got = ops.token_log_probs(many, tokens.reshape(1, 3, 2, 2))
    close(got.reshape(3, 4), want, lp_tol)
    single = ops.token_log_probs(whole[0, 4].detach(), tokens[0, 0])
    close(single, want[0, 0], lp_tol[0, 0])


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("vocab", [70, 3001])
def test_log_probs_masked_vocabulary(device, dtype, vocab):
    """-inf and the lowest value in masked columns, rows of nothing else, NaN
    in ignored rows and under a zero upstream gradient."""
    g = gen(vocab)
    low = torch.finfo(dtype).min
    logits = torch.randn(7, vocab, generator=g)
    logits[0, vocab // 2:] = -math.inf
    logits[1, : vocab // 3] = low
    logits[2] = low                   # uniform
    logits[3] = -math.inf             # no distribution: NaN
    logits[4] = math.nan              # ignored
    logits[5] = math.nan              # its upstream gradient is 0
    logits = logits.to(dtype).to(device).requires_grad_()
    tokens = torch.tensor([1, vocab - 1, 3, 0, -100, 2, 5], device=device)
    upstream = torch.tensor([1.0, -2.0, 0.5, 1.0, 1.0, 0.0, 3.0], device=device)
    lp = ops.token_log_probs(logits, tokens)
    got = lp.detach().cpu().double()
    assert got[3].isnan() and got[5].isnan() and got[4] == 0
    assert abs(got[2] + math.log(vocab)) < 64 * U * math.log(vocab)
    rest = [0, 1, 6]
    want, dwant, gg, p, z = log_probs_oracle(logits[rest], tokens[rest], 1.0, -100, upstream[rest])
    close(lp[rest], want, U * (6 * 40 + vocab / 64 + 64))
    if device == "cpu":
        return  # log_softmax's own backward knows no masked rows
    (grad,) = torch.autograd.grad(lp, logits, upstream)
    grad = grad.cpu()
    assert (grad[4] == 0).all() and (grad[5] == 0).all()
    assert grad[3].isnan().all()
    close(grad[rest], dwant, half_step(dwant, dtype) * 1.01 + gg.abs() * U * (6 * 40 + vocab / 64 + 64))
    uniform = torch.full((vocab,), -0.5 / vocab, dtype=torch.float64)
    uniform[3] += 0.5
    close(grad[2], uniform, half_step(uniform, dtype) * 1.01 + U * 64)


@pytest.mark.parametrize("device", DEVICES)
def test_log_probs_ignored_rows_pass_nothing_back(device):
    logits = torch.randn(3, 2, 40, generator=gen(1))
    logits[1, 0] = math.nan
    logits[2] = math.inf
    logits = logits.to(device).requires_grad_()
    tokens = torch.tensor([[3, 39], [7, 0], [7, 7]], device=device)
    lp = ops.token_log_probs(logits, tokens, ignore_index=7)
    (grad,) = torch.autograd.grad(lp.sum(), logits)
    assert (lp[tokens == 7] == 0).all() and lp.isfinite().all()
    assert (grad[tokens == 7] == 0).all() and grad.isfinite().all()


@pytest.mark.parametrize("device", DEVICES)
def test_log_probs_tokens_out_of_range(device):
    logits = torch.randn(4, 9, generator=gen(0)).to(device)
    tokens = torch.tensor([-1, 9, 2 ** 40, 3], device=device)
    lp = ops.token_log_probs(logits, tokens)
    assert lp[:3].isnan().all() and lp[3].isfinite()
    lp = ops.token_log_probs(logits, tokens, ignore_index=-1)
    assert lp[0] == 0 and lp[1:3].isnan().all()


@pytest.mark.parametrize("device", DEVICES)
def test_log_probs_empty(device):
    logits = torch.zeros(0, 5, 7, device=device, requires_grad=True)
    lp = ops.token_log_probs(logits, torch.zeros(0, 5, dtype=torch.long, device=device))
    assert lp.shape == (0, 5)
    (grad,) = torch.autograd.grad(lp.sum(), logits)
    assert grad.shape == logits.shape


@pytest.mark.parametrize("device", DEVICES)
def test_log_probs_gradient_against_differences(device):
    """Central differences of step h in float32: the third derivative (below 1
    in softmax) leaves h^2 / 6, the rounding of lp leaves 2 * 16 u |lp| / h."""
    g = gen(9)
    logits = torch.randn(3, 12, generator=g).to(device).requires_grad_()
    tokens = torch.tensor([0, 5, 11], device=device)
    (grad,) = torch.autograd.grad(ops.token_log_probs(logits, tokens, temperature=0.8).sum(), logits)
    h = 2.0 ** -7
    for i in range(3):
        for j in range(12):
            up, down = logits.detach().clone(), logits.detach().clone()
            up[i, j] += h
            down[i, j] -= h
            d = (ops.token_log_probs(up, tokens, temperature=0.8)[i]
                 - ops.token_log_probs(down, tokens, temperature=0.8)[i]) / (2 * h)
            assert abs(float(d - grad[i, j])) < h * h / 6 / 0.8 ** 3 + 32 * U * 10 / h


@pytest.mark.parametrize("device", DEVICES)
def test_log_probs_refusals(device):
    logits = torch.zeros(2, 5, device=device)
    tokens = torch.zeros(2, dtype=torch.long, device=device)
    with pytest.raises(TypeError, match="logits must be"):
        ops.token_log_probs(logits.double(), tokens)
    with pytest.raises(TypeError, match="tokens must be"):
        ops.token_log_probs(logits, tokens.float())
    with pytest.raises(ValueError, match="shape of logits"):
        ops.token_log_probs(logits, tokens[:1])
    with pytest.raises(ValueError, match="vocabulary"):
        ops.token_log_probs(logits[:, :0], tokens)
    for bad in (0.0, -1.0, math.inf, math.nan, 1e-40):
        with pytest.raises(ValueError, match="temperature"):
            ops.token_log_probs(logits, tokens, temperature=bad)
    if device == "cuda":
        with pytest.raises(ValueError, match="tokens is on"):
            ops.token_log_probs(logits, tokens.cpu())


@pytest.mark.parametrize("device", DEVICES)
def test_log_probs_second_derivative(device):
    """A product of the Hessian with a vector, and the gradient's derivative by
    the upstream one, an ignored place, a NaN row without upstream among them."""
    g = gen(12)
    logits = torch.randn(5, 37, generator=g) * 2
    tokens = torch.randint(0, 37, (5,), generator=g)
    tokens[1] = -100
    upstream, vec = torch.randn(5, generator=g), torch.randn(5, 37, generator=g)

    def products(x, up, at, v, call):
        x, up = x.requires_grad_(), up.requires_grad_()
        (first,) = torch.autograd.grad(call(x, at), x, up, create_graph=True)
        return (first, *torch.autograd.grad((first * v).sum(), (x, up)))

    def plain(x, at):
        lp = (x / 1.7).log_softmax(-1).gather(-1, at.clamp(min=0)[:, None]).squeeze(-1)
        return torch.where(at == -100, 0.0, lp)

    got = products(logits.to(device), upstream.to(device), tokens.to(device), vec.to(device),
                   lambda x, at: ops.token_log_probs(x, at, temperature=1.7))
    want = products(logits.double(), upstream.double(), tokens, vec.double(), plain)
    for a, b in zip(got, want):
        # sums over 37 products of terms up to 5, some 100 roundings
        assert (a.detach().cpu().double() - b.detach()).abs().max() <= 100 * U * 5 * 5
    if device == "cuda":
        x = logits.cuda()
        x[3] = math.nan
        up = upstream.cuda()
        up[3] = 0
        first = products(x, up, tokens.cuda(), vec.cuda(), lambda x, at: ops.token_log_probs(x, at))[0]
        assert (first[3] == 0).all() and (first[1] == 0).all() and first.isfinite().all()


# --------------------------------------------------------------------------- #
# token_policy_loss
# --------------------------------------------------------------------------- #
def policy_oracle(lp, old, adv, w, ref, low, high, variant, kl_c, ent_c, reduction):
    lp = lp.detach().cpu().double().requires_grad_()
    old = old.cpu().double()
    adv = adv.cpu().double().expand(lp.shape)
    w = torch.ones_like(lp) if w is None else w.cpu().double()
    keep = w != 0
    x = (lp - old)[keep]
    r = x.exp()
    c = r.clamp(1 - low, 1 + high)
    a, ww = adv[keep], w[keep]
    gain = torch.minimum(r * a, c * a) if variant == "clip" else c.detach() * x * a
    count = max(1.0, float(w.sum())) if reduction == "mean" else 1.0
    obj = -(gain * ww).sum() / count
    kl = torch.zeros((), dtype=torch.float64)
    ysize = kl
    if ref is not None:
        y = (ref.cpu().double() - lp)[keep]
        kl = ((y.expm1() - y) * ww).sum() / count
        ysize = ((y.exp() + 1 + y.abs()) * ww.abs()).detach()
    ent = ent_c * (lp[keep] * ww).sum() / count
    total = obj + kl_c * kl + ent
    (grad,) = torch.autograd.grad(total, lp)
    every = (lp.detach() - old).exp()
    out = dict(loss_total=total, loss_objective=obj, loss_kl=kl_c * kl, loss_entropy=ent, kl=kl,
               clip_fraction=((every - 1).abs() > low).double().mean(),
               ess=every.sum() ** 2 / (every ** 2).sum().clamp(min=1e-9) / every.numel(), grad=grad)
    size = dict(gain=float((gain * ww).detach().abs().sum() / count),
                kl=float(ysize.sum() / count) if ref is not None else 0.0,
                x=float(x.detach().abs().max()) if x.numel() else 0.0)
    # what a gradient's terms come to, one by one
    terms = torch.zeros_like(lp.detach())
    terms[keep] = (r * a).abs().detach() + (c * a).abs().detach() + abs(ent_c)
    if ref is not None:
        terms[keep] += abs(kl_c) * ysize / ww.abs()
    return {k: v.detach() for k, v in out.items()}, size, terms * w.abs() / count


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", [(1, 1), (3, 5), (16, 45), (1, 4099), (130, 257)])
@pytest.mark.parametrize("variant,high,kl,ent,reduction,masked", [
    ("clip", 0.2, 0.0, 0.0, "mean", "bool"),
    ("clip", 0.28, 0.05, 0.01, "mean", "int64"),
    ("cispo", 0.2, 0.02, 0.0, "sum", "float"),
    ("clip", 0.2, 0.1, 0.0, "sum", None),
])
def test_policy_loss_and_gradient(device, dtype, shape, variant, high, kl, ent, reduction, masked):
    g = gen(shape[1])
    old = (-torch.randn(shape, generator=g).abs() * 2).to(dtype)
    lp = (old.float() + 0.3 * torch.randn(shape, generator=g)).to(dtype)
    ref = (old.float() + 0.3 * torch.randn(shape, generator=g)).to(dtype) if kl else None
    adv = torch.randn(shape[0], 1, generator=g)
    mask = None
    if masked:
        mask = torch.rand(shape, generator=g) < 0.7
        if masked == "int64":
            mask = mask.long()
        elif masked == "float":
            mask = mask * torch.rand(shape, generator=g)
    move = lambda t: None if t is None else t.to(device)  # noqa: E731
    leaf = lp.to(device).requires_grad_()
    out = ops.token_policy_loss(
        leaf, move(old), move(adv), move(mask), move(ref), clip_low=0.2, clip_high=high,
        variant=variant, kl_coeff=kl, entropy_coeff=ent, reduction=reduction)
    (grad,) = torch.autograd.grad(out.loss_total, leaf)
    want, size, terms = policy_oracle(lp, old, adv, mask, ref, 0.2, high, variant, kl, ent, reduction)
    # an element is off by u |x| through its exponent and by a few roundings;
    # a sum in float32 (the CPU form) rounds log2(n) times on the way
    n = lp.numel()
    step = U * (8 + 2 * size["x"] + (0 if device == "cuda" else 2 * math.log2(n + 1) + 8))
    lp_mean = float((lp.detach().double().abs() * (1 if mask is None else mask.double().abs())).sum()) / (
        1.0 if reduction == "sum" else max(1.0, float(n if mask is None else mask.sum())))
    near = dict(loss_objective=step * size["gain"], kl=step * size["kl"],
                loss_entropy=step * abs(ent) * lp_mean, clip_fraction=U, ess=4 * step)
    near["loss_kl"] = kl * near["kl"]
    near["loss_total"] = near["loss_objective"] + near["loss_kl"] + near["loss_entropy"]
    for name, tol in near.items():
        got = float(getattr(out, name).detach())
        ref_v = float(want[name])
        assert abs(got - ref_v) <= 2 * tol + 2 * U * abs(ref_v), (name, got, ref_v)
    close(grad, want["grad"], 1.01 * half_step(want["grad"], dtype) + 2 * step * terms)
    with torch.no_grad():
        again = ops.token_policy_loss(
            leaf, move(old), move(adv), move(mask), move(ref), clip_low=0.2, clip_high=high,
            variant=variant, kl_coeff=kl, entropy_coeff=ent, reduction=reduction)
    assert all(torch.equal(a, b) for a, b in zip(again, out))


@pytest.mark.parametrize("device", DEVICES)
def test_policy_loss_separate_gradients_and_layouts(device):
    """Each differentiable output by itself; strided and mixed-type operands;
    more than two dims."""
    g = gen(5)
    wide = torch.randn(2, 3, 2 * 10, generator=g)
    lp = (-wide[..., ::2].abs()).to(device)
    old = (lp.cpu() + 0.2 * torch.randn(2, 3, 10, generator=g)).bfloat16().to(device)
    ref = (lp.cpu() + 0.2 * torch.randn(3, 2, 10, generator=g).transpose(0, 1)).to(device)
    adv = torch.randn(3, 1, generator=g).to(device)
    mask = (torch.rand(10, 3, 2, generator=g) < 0.6).permute(2, 1, 0).to(device)
    for pick in ("loss_objective", "loss_kl", "loss_entropy"):
        leaf = lp.clone().requires_grad_()
        out = ops.token_policy_loss(leaf, old, adv, mask, ref, kl_coeff=0.1, entropy_coeff=0.3)
        (grad,) = torch.autograd.grad(3.0 * getattr(out, pick), leaf)
        ref_leaf = lp.double().cpu().requires_grad_()
        x = ref_leaf - old.double().cpu()
        r = x.exp()
        a = adv.double().cpu()
        y = ref.double().cpu() - ref_leaf
        term = {"loss_objective": -torch.minimum(r * a, r.clamp(0.8, 1.2) * a),
                "loss_kl": 0.1 * (y.expm1() - y), "loss_entropy": 0.3 * ref_leaf}[pick]
        keep = mask.cpu()
        (want,) = torch.autograd.grad(3.0 * term[keep].sum() / keep.sum(), ref_leaf)
        close(grad, want, 64 * U * (want.abs() + 3.0 / float(keep.sum())))


@pytest.mark.parametrize("device", DEVICES)
def test_policy_loss_masked_places_hold_anything(device):
    lp = torch.tensor([[-1.0, math.nan, -2.0, math.inf]], device=device, requires_grad=True)
    old = torch.tensor([[-1.1, -math.inf, -2.0, math.nan]], device=device)
    ref = torch.tensor([[-0.9, math.nan, -2.5, -math.inf]], device=device)
    mask = torch.tensor([[True, False, True, False]], device=device)
    out = ops.token_policy_loss(lp, old, torch.ones(1, 1, device=device), mask, ref, kl_coeff=0.1)
    (grad,) = torch.autograd.grad(out.loss_total, lp)
    assert out.loss_total.isfinite() and grad.isfinite().all()
    assert grad[0, 1] == 0 and grad[0, 3] == 0 and (grad[0, ::2] != 0).all()
    nothing = ops.token_policy_loss(lp, old, torch.ones(1, 1, device=device),
                                    torch.zeros_like(mask), ref, kl_coeff=0.1)
    assert nothing.loss_total == 0 and nothing.kl == 0
    (grad,) = torch.autograd.grad(nothing.loss_total, lp)
    assert (grad == 0).all()


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("mask_dtype", [torch.bool, torch.uint8, torch.int8, torch.int16, torch.int32, torch.int64,
                                        torch.float16, torch.bfloat16, torch.float32, torch.float64])
@pytest.mark.parametrize("shape", [(3, 8), (7, 5), (130, 257)])
def test_policy_loss_mask_types(device, mask_dtype, shape):
    """Weights 0, 1 and, where the type has them, 2 and -1: sums of float32
    terms of size 10, each off by some 16 u."""
    g = gen(31)
    old = -torch.rand(shape, generator=g) * 2
    lp = old + 0.3 * torch.randn(shape, generator=g)
    adv = torch.randn(shape[0], 1, generator=g)
    mask = torch.randint(0 if mask_dtype in (torch.bool, torch.uint8) else -1, 3, shape, generator=g).to(mask_dtype)
    x = lp.to(device).requires_grad_()
    out = ops.token_policy_loss(x, old.to(device), adv.to(device), mask.to(device), reduction="sum",
                                entropy_coeff=0.1)
    (grad,) = torch.autograd.grad(out.loss_total, x)
    want, _, _ = policy_oracle(lp, old, adv, mask, None, 0.2, 0.2, "clip", 0.0, 0.1, "sum")
    n = lp.numel()
    assert abs(float(out.loss_total.detach()) - float(want["loss_total"])) <= 16 * U * 10 * n
    close(grad, want["grad"], 64 * U * (want["grad"].abs() + 1))


@pytest.mark.parametrize("device", DEVICES)
def test_policy_loss_outputs_change_in_place(device):
    lp = torch.zeros(2, 3, device=device, requires_grad=True)
    out = ops.token_policy_loss(lp, torch.zeros(2, 3, device=device), torch.ones(2, 1, device=device))
    total = out.loss_total
    kept = float(out.loss_objective.detach())
    total += 1.0
    assert float(out.loss_objective.detach()) == kept
    total.backward()
    assert torch.allclose(lp.grad, torch.full_like(lp, -1 / 6))


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("grad", [False, True])
def test_policy_loss_outputs_are_each_their_own(device, grad):
    """Absent terms too: a change of one in place leaves the others."""
    lp = torch.zeros(2, 3, device=device, requires_grad=grad)
    out = ops.token_policy_loss(lp, torch.zeros(2, 3, device=device), torch.ones(2, 1, device=device))
    for i in range(7):
        before = [float(x.detach()) for x in out]
        out[i].detach().add_(1.0)
        after = [float(x.detach()) for x in out]
        assert after == [x + (j == i) for j, x in enumerate(before)]


@pytest.mark.parametrize("device", DEVICES)
def test_policy_loss_refusals(device):
    lp = torch.zeros(2, 3, device=device)
    adv = torch.zeros(2, 1, device=device)

    def call(a=lp, b=lp, c=adv, **kw):
        return ops.token_policy_loss(a, b, c, kw.pop("mask", None), kw.pop("ref", None), **kw)

    with pytest.raises(TypeError, match="log_probs must be"):
        call(a=lp.double(), b=lp)
    with pytest.raises(ValueError, match="old_log_probs must have"):
        call(b=lp[:1])
    with pytest.raises(ValueError, match="does not broadcast"):
        call(c=torch.zeros(3, 1, device=device))
    with pytest.raises(ValueError, match="mask must have"):
        call(mask=torch.ones(2, device=device))
    with pytest.raises(TypeError, match="unsupported dtype"):
        call(mask=torch.ones(2, 3, dtype=torch.complex64, device=device))
    with pytest.raises(ValueError, match="must not require"):
        call(b=lp.clone().requires_grad_())
    with pytest.raises(ValueError, match="must not require"):
        call(c=adv.clone().requires_grad_())
    with pytest.raises(ValueError, match="empty"):
        call(a=lp[:, :0], b=lp[:, :0])
    with pytest.raises(ValueError, match="clip_low"):
        call(clip_low=-0.1)
    with pytest.raises(ValueError, match="coeff"):
        call(kl_coeff=math.nan)
    with pytest.raises(ValueError, match="variant"):
        call(variant="ppo")
    with pytest.raises(ValueError, match="reduction"):
        call(reduction="none")


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape,shift", [((1, 1), 0.0), ((5, 33), 0.0), ((5, 33), 60.0), ((5, 33), -12.0),
                                         ((130, 257), 0.0)])
@pytest.mark.parametrize("dense", [False, True])
def test_policy_loss_ess_gradient(device, dtype, shape, shift, dense):
    """Alone and with the loss's, masked places among them; ratios so large that
    their squares leave float32, and so small that the sum meets its floor."""
    g = gen(14)
    old = (-torch.rand(shape, generator=g) * 2).to(dtype)
    lp = (old.float() + shift + 0.4 * torch.randn(shape, generator=g)).to(dtype)
    adv = torch.randn(shape, generator=g)
    mask = torch.rand(shape, generator=g) < 0.6
    x = lp.to(device)
    if not dense:
        x = x.t().contiguous().t()
    x.requires_grad_()
    out = ops.token_policy_loss(x, old.to(device), adv.to(device), mask.to(device))
    y = lp.double().requires_grad_()
    r = (y - old.double()).exp()
    ess = r.sum() ** 2 / (r ** 2).sum().clamp(min=1e-9) / r.numel()
    (want,) = torch.autograd.grad(ess, y)
    if device == "cpu" and shift == 60.0:
        return  # elementary float32 overflows here
    (got,) = torch.autograd.grad(1.5 * out.ess, x, retain_graph=True)
    t = (r * r.sum() / (r ** 2).sum().clamp(min=1e-9)).detach()
    size = 1.5 * 2 / r.numel() * (t + t * t)
    # the exponent's argument is off by u of its size, up to some 100 in base 2;
    # float32 sums on the CPU add their length's root
    tol = size * U * 400 * (4 if device == "cpu" else 1) + 1.5 * want.abs() * torch.finfo(dtype).eps / 2 + 1e-30
    tiny = torch.finfo(dtype).smallest_normal
    assert ((got.cpu().double() - 1.5 * want).abs() <= tol + tiny).all()
    if shift == 0.0:
        (both,) = torch.autograd.grad(1.5 * out.ess + out.loss_total, x, retain_graph=True)
        (loss,) = torch.autograd.grad(out.loss_total, x)
        assert ((both - got - loss).abs().double().cpu()
                <= 3 * torch.finfo(dtype).eps * (got.abs() + loss.abs()).double().cpu() + tiny).all()


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("variant", ["clip", "cispo"])
@pytest.mark.parametrize("reduction", ["mean", "sum"])
def test_policy_loss_second_derivative(device, variant, reduction):
    """The gradient's derivative by the log-probs and by the upstream gradients
    of all five scalars; a masked place is far off."""
    g = gen(13)
    old = -torch.rand(4, 9, generator=g) * 2
    lp = old + 0.3 * torch.randn(4, 9, generator=g)
    adv, ref = torch.randn(4, 1, generator=g), old + 0.2 * torch.randn(4, 9, generator=g)
    mask = torch.rand(4, 9, generator=g) < 0.8
    mask[0, 0] = False
    vec = torch.randn(4, 9, generator=g)
    conf = dict(clip_high=0.28, kl_coeff=0.3, entropy_coeff=0.1)

    def products(scalars, lp, v):
        assert len(scalars) == 5
        ups = [torch.tensor(u, dtype=lp.dtype, device=lp.device, requires_grad=True)
               for u in (0.7, -1.1, 0.4, 2.0, 1.3)]
        (first,) = torch.autograd.grad(scalars, lp, ups, create_graph=True)
        return (first, *torch.autograd.grad((first * v).sum(), (lp, *ups)))

    lp[0, 0] = old[0, 0] - 9.0
    x = lp.to(device).requires_grad_()
    out = ops.token_policy_loss(x, old.to(device), adv.to(device), mask.to(device), ref.to(device),
                                variant=variant, reduction=reduction, **conf)
    got = products((*out[:4], out.ess), x, vec.to(device))

    y = lp.double().requires_grad_()
    w = mask.double()
    r = (y - old.double()).exp()
    c = r.clamp(0.8, 1.28)
    a = adv.double()
    gain = torch.minimum(r * a, c * a) if variant == "clip" else c.detach() * (y - old.double()) * a
    n = w.sum() if reduction == "mean" else 1.0
    d = ref.double() - y
    obj, kl, ent = -(gain * w).sum() / n, 0.3 * ((d.exp() - 1 - d) * w).sum() / n, 0.1 * (y * w).sum() / n
    ess = r.sum() ** 2 / (r ** 2).sum() / r.numel()
    want = products((obj + kl + ent, obj, kl, ent, ess), y, vec.double())
    for a, b in zip(got, want):
        # terms up to some 20 (e^9 of the masked one has weight 0), 36 of them in a
        # sum, 40 roundings each
        size = 20 * (1 if reduction == "mean" else 36)
        assert (a.detach().cpu().double() - b.detach()).abs().max() <= 40 * U * size

    x = lp.clone()
    x[0, 0] = math.nan  # masked: nothing of it comes back without the ess
    x = x.to(device).requires_grad_()
    total = ops.token_policy_loss(x, old.to(device), adv.to(device), mask.to(device), ref.to(device),
                                  variant=variant, reduction=reduction, **conf).loss_total
    (first,) = torch.autograd.grad(total, x, create_graph=True)
    assert first.isfinite().all() and first[0, 0] == 0


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dense", [True, False])
def test_policy_loss_kl_gradient_far_from_the_reference(device, dtype, dense):
    """1 - e^y, y = ref - log_prob: -1 (times the coefficient) for a reference
    that rules the token out, by infinity or the lowest value.  The exponent's
    argument is off by u of its size, and two more roundings."""
    low = torch.finfo(dtype).min
    y = torch.tensor([-math.inf, low, -1e9, -3.5e7, -90.0, -30.0, -17.0, -5.0, -0.75, -0.5, 0.25, 0.5, 0.75, 5.0, 9.0])
    ref = y.to(dtype)[None].repeat(3, 1)
    old = torch.zeros_like(ref)
    lp = torch.zeros_like(ref).to(device)
    if not dense:
        lp = lp.t().contiguous().t()
    lp.requires_grad_()
    out = ops.token_policy_loss(lp, old.to(device), torch.ones(3, 1, device=device), None, ref.to(device),
                                kl_coeff=0.5, reduction="sum")
    (grad,) = torch.autograd.grad(out.loss_kl, lp, retain_graph=True)
    want = -0.5 * torch.expm1(ref.double())
    tol = 0.5 * U * (ref.double().exp() * (4 + 3 * ref.double().abs().clamp(max=100)) + 4)
    close(grad, want, tol + 1.01 * half_step(want, dtype))
    # and as part of the whole: the objective's is -1
    (grad,) = torch.autograd.grad(out.loss_total, lp)
    close(grad, want - 1, tol + 4 * U + 1.01 * half_step(want - 1, dtype))


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("create_graph", [False, True])
def test_policy_loss_terms_without_weight_are_left_out(device, create_graph):
    """A term whose coefficient is 0 does not count, infinite or not; kl is still
    reported, and every loss still has a gradient."""
    old = torch.tensor([[-1.0, -2.0, -1.5]], device=device)
    ref = torch.tensor([[-math.inf, math.inf, -1.0]], device=device)
    adv = torch.ones(1, 1, device=device)

    def grad(loss, lp):
        return torch.autograd.grad(loss, lp, create_graph=create_graph, retain_graph=True)[0].detach()

    lp = (old + 0.1).requires_grad_()
    out = ops.token_policy_loss(lp, old, adv, None, ref, entropy_coeff=0.25)
    assert not out.kl.isfinite() and out.loss_kl == 0  # inf - inf
    assert abs(float(out.loss_total.detach() - out.loss_objective.detach() - out.loss_entropy.detach())) <= 4 * U
    want = (0.25 - (lp.detach() - old).exp()) / 3
    assert ((grad(out.loss_total, lp) - want).abs() <= 16 * U).all()
    assert (grad(out.loss_kl, lp) == 0).all()
    # no reference at all, and a log-prob of -inf without an entropy term
    lp = torch.tensor([[-1.0, -math.inf, -1.5]], device=device, requires_grad=True)
    out = ops.token_policy_loss(lp, old, adv)
    assert out.loss_entropy == 0 and out.loss_kl == 0 and out.kl == 0
    assert out.loss_total == out.loss_objective and out.loss_total.isfinite()
    want = torch.tensor([[-1.0, 0.0, -1.0]], device=device) / 3
    assert ((grad(out.loss_total, lp) - want).abs() <= 16 * U).all()
    assert (grad(out.loss_kl, lp) == 0).all() and (grad(out.loss_entropy, lp) == 0).all()


# --------------------------------------------------------------------------- #
# the paged cache
# --------------------------------------------------------------------------- #
def make_cache(g, batch, columns, kv_heads, page, dim, dtype, device, spare=2):
    """A cache whose free pages and slots hold NaN, and a shuffled table."""
    pages = batch * columns + spare
    k = torch.full((pages, kv_heads, page, dim), math.nan)
    table = torch.randperm(pages, generator=g)[: batch * columns].reshape(batch, columns).int()
    return k.to(dtype).to(device), k.clone().to(dtype).to(device), table.to(device)


def rotate64(x, cos, sin, interleaved):
    """[T, H, D] by [T, R / 2] as complex numbers."""
    half = cos.shape[-1]
    one = slice(0, 2 * half, 2) if interleaved else slice(0, half)
    two = slice(1, 2 * half, 2) if interleaved else slice(half, 2 * half)
    y = x.clone()
    z = torch.complex(x[..., one], x[..., two]) * torch.complex(cos, sin).unsqueeze(1)
    y[..., one], y[..., two] = z.real, z.imag
    return y


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("batch,width,heads,kv_heads,dim,page,rotary,interleaved,odd", [
    (3, 1, 4, 4, 64, 16, 0, False, False),
    (3, 1, 8, 2, 128, 8, 128, False, False),
    (2, 7, 12, 4, 80, 4, 80, True, False),
    (2, 19, 5, 1, 96, 16, 48, False, False),
    (4, 5, 6, 3, 80, 1, 40, False, False),
    (2, 9, 4, 2, 80, 16, 40, True, False),
    (2, 9, 7, 1, 24, 16, 8, False, False),
    (2, 33, 16, 2, 256, 32, 256, True, False),
    (3, 6, 3, 3, 40, 8, 20, True, True),
    (3, 6, 2, 1, 8, 64, 8, False, True),
    (1, 3, 40, 40, 64, 16, 2, False, False),
])
def test_append(device, dtype, batch, width, heads, kv_heads, dim, page, rotary, interleaved, odd):
    g = gen(dim + width)
    past = 11
    columns = -(-(past + width) // page)
    k_cache, v_cache, table = make_cache(g, batch, columns, kv_heads, page, dim, dtype, device)
    # views of one projection; `odd` shifts them off every alignment
    rows = torch.randn(batch, width, (heads + 2 * kv_heads) * dim + 1, generator=g).to(dtype).to(device)
    rows = rows[..., 1:] if odd else rows[..., :-1].contiguous()
    q, k, v = rows.split([heads * dim, kv_heads * dim, kv_heads * dim], -1)
    q, k, v = (t.unflatten(-1, (-1, dim)) for t in (q, k, v))
    start = torch.randint(0, past, (batch,), generator=g)
    lengths = torch.randint(0, width + 1, (batch,), generator=g)
    lengths[0] = width
    if batch > 2:
        lengths[1] = 0
    rope = ops.rotary_table(past + width, rotary, device=device) if rotary else None
    got_q = ops.paged_kv_append(
        k, v, k_cache, v_cache, table, start.to(device).int(), lengths=lengths.to(device),
        q=q if rotary else None, rope=rope, interleaved=interleaved)
    assert (got_q is None) == (rotary == 0)
    want_k = torch.full(k_cache.shape, math.nan, dtype=torch.float64)
    want_v, size = want_k.clone(), want_k.clone()
    want_q = torch.zeros(q.shape, dtype=torch.float64)
    for b in range(batch):
        n, first = int(lengths[b]), int(start[b])
        kk, qq = k[b, :n].cpu().double(), q[b, :n].cpu().double()
        if rotary:
            cos, sin = (t[first:first + n].cpu().double() for t in rope)
            kk, qq = (rotate64(t, cos, sin, interleaved) for t in (kk, qq))
            want_q[b, :n] = qq
        place = torch.arange(first, first + n)
        at = table[b].cpu().long()[place // page]
        want_k[at, :, place % page] = kk
        want_v[at, :, place % page] = v[b, :n].cpu().double()
    # two products and a sum in float32, each rounded, then the cache's rounding
    worst = float(rows.abs().max()) * 4 * U
    close(v_cache, want_v, 0.0)
    close(k_cache, want_k, 1.01 * half_step(want_k, dtype) + worst if rotary else 0.0)
    if rotary:
        close(got_q, want_q, 1.01 * half_step(want_q, dtype) + worst)


@pytest.mark.parametrize("device", DEVICES)
def test_append_is_an_in_place_change(device):
    """A cache that an earlier operation keeps for its backward pass: the
    backward pass refuses, as after any other change in place.  Inference
    tensors, which have no version, are written as before."""
    def case():
        k_cache = torch.zeros(4, 1, 8, 16, device=device)
        return k_cache, torch.zeros_like(k_cache), torch.ones(2, 1, 1, 16, device=device)

    table = torch.tensor([[1], [3]], dtype=torch.int32, device=device)
    start = torch.zeros(2, dtype=torch.int32, device=device)
    for which in (0, 1):
        caches = case()
        w = torch.ones((), device=device, requires_grad=True)
        loss = (w * caches[which]).sum()
        ops.paged_kv_append(caches[2], caches[2], caches[0], caches[1], table, start)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            loss.backward()
    with torch.inference_mode():
        k_cache, v_cache, k = case()
        ops.paged_kv_append(k, k, k_cache, v_cache, table, start)
        assert (k_cache[1, 0, 0] == 1).all() and (k_cache[0] == 0).all()


@pytest.mark.parametrize("device", DEVICES)
def test_append_bad_places_write_nothing(device):
    g = gen(1)
    k_cache, v_cache, _ = make_cache(g, 6, 1, 2, 8, 16, torch.float32, device)
    before = k_cache.clone()
    table = torch.tensor([[-1], [8], [2 ** 31 - 1], [2], [3], [4]], dtype=torch.int32, device=device)
    assert k_cache.shape[0] == 8
    start = torch.tensor([0, 0, 0, -2, 7, 2 ** 33], device=device)
    k = torch.randn(6, 2, 2, 16, generator=g).to(device)
    ops.paged_kv_append(k, k, k_cache, v_cache, table, start)
    before[3, :, 7] = k[4, 0]
    assert torch.equal(k_cache.isnan(), before.isnan())
    assert torch.equal(k_cache.nan_to_num(), before.nan_to_num())
    empty = torch.zeros(6, 0, dtype=torch.int32, device=device)
    ops.paged_kv_append(k, k, k_cache, v_cache, empty, start)
    ops.paged_kv_append(k[:0], k[:0], k_cache, v_cache, table[:0], start[:0])
    ops.paged_kv_append(k[:, :0], k[:, :0], k_cache, v_cache, table, start)
    assert torch.equal(k_cache.nan_to_num(), before.nan_to_num())
    # past the rotation's table: NaN, not what lies behind it
    rope = ops.rotary_table(3, 16, device=device)
    zero = torch.zeros(6, dtype=torch.int32, device=device)
    good = torch.arange(6, dtype=torch.int32, device=device)[:, None]
    wide = k.repeat(1, 2, 1, 1)
    q = ops.paged_kv_append(wide, wide, k_cache, v_cache, good, zero, q=wide, rope=rope)
    assert q[:, :3].isfinite().all() and q[:, 3].isnan().all()
    assert k_cache[:6, :, :3].isfinite().all() and k_cache[:6, :, 3].isnan().all()


def attend_oracle(q, k_cache, v_cache, table, lengths, scale):
    q, k_cache, v_cache = (t.cpu().double() for t in (q, k_cache, v_cache))
    table = table.cpu().long()
    batch, heads, dim = q.shape
    kv_heads, page = k_cache.shape[1:3]
    out, tol = torch.zeros_like(q), torch.zeros_like(q)
    for b in range(batch):
        n = min(int(lengths[b]), table.shape[1] * page)
        place = torch.arange(max(0, n))
        at = table[b][place // page] if n > 0 else place
        keep = (at >= 0) & (at < k_cache.shape[0])
        place, at = place[keep], at[keep]
        if not len(place):
            continue
        for h in range(heads):
            kv = h // (heads // kv_heads)
            k, v = k_cache[at, kv, place % page], v_cache[at, kv, place % page]
            score = (k @ q[b, h]) * scale
            p = torch.softmax(score, 0)
            out[b, h] = p @ v
            # a score of dim products adds up in float32 (the matrix unit may cut
            # instead of rounding: 2 u each); exp turns its error into a relative
            # one; weights enter the second product in two 16-bit parts (2^-16);
            # the sums over n keys round n times at most
            off = float(((k.abs() @ q[b, h].abs()) * abs(scale)).max()) * 2 * U * (dim + 8)
            rel = 2 * off + 2.0 ** -16 + 2 * U * (len(place) + 16)
            tol[b, h] = rel * (p @ v.abs())
    return out, tol


def fill_cache(g, cache, table, lengths):
    """Random keys or values in the slots that sequences hold; NaN elsewhere."""
    page = cache.shape[2]
    for b in range(table.shape[0]):
        n = min(int(lengths[b]), table.shape[1] * page)
        if n <= 0:
            continue
        place = torch.arange(n)
        at = table[b].cpu().long()[place // page]
        cache[at, :, place % page] = torch.randn(n, cache.shape[1], cache.shape[3], generator=g).to(
            cache.dtype).to(cache.device)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("lengths,heads,kv_heads,dim,page", [
    ([1], 1, 1, 64, 16),
    ([0, 1, 2, 17], 4, 4, 64, 16),
    ([31, 32, 33, 64, 65], 8, 2, 128, 8),
    ([100, 7], 14, 2, 80, 4),
    ([257, 0, 300], 12, 12, 64, 16),
    ([1000], 5, 1, 96, 1),
    ([511, 513, 129], 32, 2, 256, 128),
    ([77, 40], 40, 1, 40, 32),
    ([33], 16, 16, 8, 2),
    ([5000, 3, 129, 2048], 32, 8, 128, 64),
    ([3000] * 3, 7, 1, 192, 256),
    ([-3, 9], 24, 1, 64, 16),
])
def test_attend(device, dtype, lengths, heads, kv_heads, dim, page):
    g = gen(sum(lengths) + dim)
    batch = len(lengths)
    columns = max(1, -(-max(lengths) // page))
    k_cache, v_cache, table = make_cache(g, batch, columns, kv_heads, page, dim, dtype, device)
    fill_cache(g, k_cache, table, lengths)
    fill_cache(g, v_cache, table, lengths)
    q = (torch.randn(batch, heads, dim, generator=g) * 2).to(dtype).to(device)
    count = torch.tensor(lengths, device=device)
    out = ops.paged_attention_decode(q, k_cache, v_cache, table, count)
    assert out.dtype == dtype and out.is_contiguous()
    want, tol = attend_oracle(q, k_cache, v_cache, table, lengths, dim ** -0.5)
    close(out, want, 1.01 * half_step(want, dtype) + tol)
    again = ops.paged_attention_decode(q, k_cache, v_cache, table, count.int(), scale=dim ** -0.5)
    assert torch.equal(again, out)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("batch,longest,heads,kv_heads,dim,page", [
    (40, 700, 16, 8, 128, 16),    # single waves as workers, items shared
    (130, 1300, 6, 3, 64, 8),     # the same, more sequences than lanes
    (90, 1500, 20, 1, 40, 64),    # workgroups, two blocks of heads
    (300, 120, 8, 4, 64, 16),     # one wave to an item
    (33, 900, 24, 8, 72, 32),     # single waves, dims past the row
])
def test_attend_batches(dtype, batch, longest, heads, kv_heads, dim, page):
    """Ragged batches of every way a call is split: lengths of 0, 1 and the
    longest among them."""
    device = "cuda"
    g = gen(batch + dim)
    lengths = torch.randint(0, longest + 1, (batch,), generator=g).tolist()
    lengths[0], lengths[batch // 2], lengths[-1] = 0, longest, 1
    k_cache, v_cache, table = make_cache(g, batch, -(-longest // page), kv_heads, page, dim, dtype, device)
    fill_cache(g, k_cache, table, lengths)
    fill_cache(g, v_cache, table, lengths)
    table[1, 0] = -1
    q = (torch.randn(batch, heads, dim, generator=g) * 2).to(dtype).to(device)
    out = ops.paged_attention_decode(q, k_cache, v_cache, table, torch.tensor(lengths, device=device))
    some = sorted({0, 1, 2, 63 % batch, 64 % batch, batch // 2, batch - 2, batch - 1})
    want, tol = attend_oracle(q[some], k_cache, v_cache, table[some], [lengths[b] for b in some], dim ** -0.5)
    close(out[some], want, 1.01 * half_step(want, dtype) + tol)
    # the others against the same sequence by itself: a row of a batch is its own
    alone = torch.cat([ops.paged_attention_decode(
        q[b:b + 1], k_cache, v_cache, table[b:b + 1], torch.tensor(lengths[b:b + 1], device=device))
        for b in range(0, batch, 7)])
    both = (out[::7].float() - alone.float()).abs()
    assert (both <= 2 * torch.finfo(dtype).eps * alone.float().abs() + 1e-3).all()


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("batch", [65535, 65536, 70001])
def test_attend_many_sequences(device, batch):
    """More sequences than a grid's second axis takes, without a page and with
    one of a few keys: a key of its own for each third sequence."""
    k_cache = torch.zeros(3, 1, 8, 8, device=device)
    k_cache[1:] = 1.0
    v_cache = torch.arange(24.0, device=device).view(3, 1, 8, 1).expand(-1, -1, -1, 8).contiguous()
    q = torch.zeros(batch, 1, 8, device=device)
    lengths = torch.arange(batch, device=device) % 3
    none = torch.zeros(batch, 0, dtype=torch.int32, device=device)
    assert (ops.paged_attention_decode(q, k_cache, v_cache, none, lengths) == 0).all()
    table = (torch.arange(batch, device=device) % 2).int()[:, None]
    out = ops.paged_attention_decode(q, k_cache, v_cache, table, lengths)
    # no key: 0; one: the page's first value; two: the mean of its first two
    want = torch.where(lengths == 0, 0.0, 8.0 * table[:, 0] + 0.5 * (lengths - 1))
    assert torch.equal(out[:, 0], want[:, None].expand(-1, 8))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("tiles", [17, 21, 33])
def test_attend_odd_workers(dtype, tiles):
    """One item shared by an odd number of workgroups (a fourth of its tiles,
    rounded up): the parts' wide accesses are aligned."""
    g = gen(tiles)
    keys = 16 if dtype == torch.float32 else 32
    n = keys * tiles - 3
    k_cache, v_cache, table = make_cache(g, 1, -(-n // 16), 1, 16, 128, dtype, "cuda")
    fill_cache(g, k_cache, table, [n])
    fill_cache(g, v_cache, table, [n])
    q = torch.randn(1, 5, 128, generator=g).to(dtype).cuda()
    out = ops.paged_attention_decode(q, k_cache, v_cache, table, torch.tensor([n], device="cuda"))
    want, tol = attend_oracle(q, k_cache, v_cache, table, [n], 128 ** -0.5)
    close(out, want, 1.01 * half_step(want, dtype) + tol)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", DTYPES)
def test_attend_bad_pages_and_layouts(device, dtype):
    """Missing pages are left out, a length past the table is cut, layer views
    of a bigger cache and strided queries and tables are read in place."""
    g = gen(8)
    batch, heads, kv_heads, dim, page, columns = 4, 6, 3, 64, 16, 5
    k_cache, v_cache, table = make_cache(g, batch, columns, kv_heads, page, dim, dtype, device)
    lengths = [columns * page] * batch
    fill_cache(g, k_cache, table, lengths)
    fill_cache(g, v_cache, table, lengths)
    layers_k, layers_v = (torch.full((2,) + t.shape[:2] + (3,) + t.shape[2:], math.nan, dtype=dtype, device=device)
                          for t in (k_cache, v_cache))
    layers_k[1, :, :, 2] = k_cache
    layers_v[1, :, :, 2] = v_cache
    wide = torch.full((batch, 2 * columns), 2 ** 30, dtype=torch.int32, device=device)
    wide[:, ::2] = table
    table = wide[:, ::2]
    table[0, 1], table[0, 4], table[1, 0] = -1, k_cache.shape[0], 2 ** 31 - 1
    table[2] = -5
    lengths = [79, 10, 80, 10 ** 9]
    q = torch.randn(batch, 2 * heads, dim + 8, generator=g).to(dtype).to(device)[:, ::2, :dim]
    out = ops.paged_attention_decode(
        q, layers_k[1, :, :, 2], layers_v[1, :, :, 2], table, torch.tensor(lengths, device=device), scale=0.3)
    want, tol = attend_oracle(q, k_cache, v_cache, table, lengths, 0.3)
    assert (want[1] == 0).all() and (want[2] == 0).all()
    close(out, want, 1.01 * half_step(want, dtype) + tol)
    odd = torch.randn(batch, heads, dim + 1, generator=g).to(dtype).to(device)[..., 1:]
    out = ops.paged_attention_decode(odd, k_cache, v_cache, table, torch.tensor(lengths, device=device))
    want, tol = attend_oracle(odd, k_cache, v_cache, table, lengths, dim ** -0.5)
    close(out, want, 1.01 * half_step(want, dtype) + tol)
    none = ops.paged_attention_decode(q, k_cache, v_cache, table[:, :0], torch.tensor(lengths, device=device))
    assert (none == 0).all()
    assert ops.paged_attention_decode(
        q[:0], k_cache, v_cache, table[:0], torch.zeros(0, dtype=torch.int32, device=device)).shape == (0, heads, dim)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_attend_one_key_dominates(device, dtype):
    """A score far above the rest, first, last or in the middle, gives that
    key's value: the others' weights are below exp(-60)."""
    g = gen(2)
    n, dim, page = 700, 64, 16
    for hot in (0, 350, 699):
        k_cache, v_cache, table = make_cache(g, 1, 44, 1, page, dim, dtype, device)
        fill_cache(g, k_cache, table, [n])
        fill_cache(g, v_cache, table, [n])
        at = int(table[0, hot // page])
        k_cache[at, 0, hot % page] = 16.0
        q = torch.full((1, 2, dim), 1.0, dtype=dtype, device=device)
        out = ops.paged_attention_decode(q, k_cache, v_cache, table, torch.tensor([n], device=device))
        assert torch.equal(out[0, 0], v_cache[at, 0, hot % page])
        assert torch.equal(out[0, 1], out[0, 0])


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("gap", [8.0, 14.0, 16.0, 17.25, 19.0])
@pytest.mark.parametrize("batch,heads,kv_heads,dim,n", [
    (2, 3, 1, 64, 61),       # one workgroup to an item
    (1, 4, 2, 128, 5000),    # items shared by workgroups
    (40, 16, 8, 128, 900),   # single waves as workers
    (1030, 1, 1, 64, 500),   # one wave to an item
])
def test_attend_small_weights_count(device, dtype, gap, batch, heads, kv_heads, dim, n):
    """A key of value 0 whose score lies ``gap`` above the others': the output
    is what the small weights bring.  float16 weights are held times 2^15 in two
    halves, so that each is off by half the smallest half, 2^-25, at most: 2^-40
    of the largest weight."""
    if device == "cpu" and batch > 2:
        pytest.skip("the CPU form has no split")
    g = gen(n)
    page = 16
    columns = -(-n // page)
    lengths = [n] * batch
    k_cache, v_cache, table = make_cache(g, batch, columns, kv_heads, page, dim, dtype, device)
    k_cache.copy_(0.01 * torch.randn(k_cache.shape, generator=g))
    v_cache.copy_(0.5 + torch.rand(v_cache.shape, generator=g))
    for b in range(batch):
        hot = (37 * b) % n
        at = int(table[b, hot // page])
        k_cache[at, :, hot % page] = 8 * gap / dim
        v_cache[at, :, hot % page] = 0
    q = torch.ones(batch, heads, dim, dtype=dtype, device=device)
    out = ops.paged_attention_decode(
        q, k_cache, v_cache, table, torch.tensor(lengths, device=device), scale=0.125)
    some = sorted({0, batch // 2, batch - 1})
    want, tol = attend_oracle(q[some], k_cache, v_cache, table[some], [n] * len(some), 0.125)
    if dtype == torch.float16:
        tol = tol + 2.0 ** -40 * n * 1.5
    close(out[some], want, 1.01 * half_step(want, dtype) + tol)


@pytest.mark.parametrize("device", DEVICES)
def test_paged_refusals(device):
    k_cache = torch.zeros(4, 2, 8, 16, device=device)
    v_cache = torch.zeros_like(k_cache)
    table = torch.zeros(3, 2, dtype=torch.int32, device=device)
    start = torch.zeros(3, dtype=torch.int32, device=device)
    k = torch.zeros(3, 1, 2, 16, device=device)
    q4, q = torch.zeros(3, 1, 4, 16, device=device), torch.zeros(3, 4, 16, device=device)
    rope = ops.rotary_table(8, 16, device=device)

    def append(k=k, v=None, kc=k_cache, vc=v_cache, t=table, s=start, **kw):
        return ops.paged_kv_append(k, k if v is None else v, kc, vc, t, s, **kw)

    def attend(q=q, kc=k_cache, vc=v_cache, t=table, n=start, **kw):
        return ops.paged_attention_decode(q, kc, vc, t, n, **kw)

    for bad, error, text in [
        (dict(k=k[0]), ValueError, "k and v must be"),
        (dict(v=k[:, :, :1]), ValueError, "k and v must be"),
        (dict(k=k.bfloat16()), TypeError, "cache's dtype"),
        (dict(kc=k_cache.double(), vc=v_cache.double()), TypeError, "share one dtype"),
        (dict(vc=v_cache.half()), TypeError, "share one dtype"),
        (dict(kc=k_cache[:, :, :6], vc=v_cache[:, :, :6]), ValueError, "power of two"),
        (dict(kc=k_cache[:, :1], vc=v_cache[:, :1]), ValueError, "expected 2 of"),
        (dict(kc=k_cache[:0], vc=v_cache[:0]), ValueError, "pages"),
        (dict(kc=k_cache.transpose(2, 3).contiguous().transpose(2, 3)), ValueError, "dense"),
        (dict(t=table.long()), TypeError, "page_table must be int32"),
        (dict(t=table[:2]), ValueError, "page_table must be"),
        (dict(s=start[:2]), ValueError, "start must be"),
        (dict(s=start.float()), TypeError, "start must be"),
        (dict(lengths=start[:2]), ValueError, "lengths must be"),
        (dict(q=q4), ValueError, "no rope"),
        (dict(q=q, rope=rope), ValueError, "q must be"),
        (dict(q=q4.half(), rope=rope), TypeError, "q must have"),
        (dict(rope=(rope[0].double(), rope[1].double())), TypeError, "rope must be float32"),
        (dict(rope=(rope[0], rope[1][:4])), ValueError, "rope must be"),
        (dict(rope=(rope[0].repeat(1, 2), rope[1].repeat(1, 2))), ValueError, "rope must be"),
        (dict(rope=(rope[0][:, ::2], rope[1][:, ::2])), ValueError, "contiguous"),
        (dict(k=k.clone().requires_grad_()), ValueError, "no_grad"),
        (dict(vc=k_cache), ValueError, "same memory"),
        (dict(kc=k_cache[:1].expand(4, -1, -1, -1)), ValueError, "expanded"),
    ]:
        with pytest.raises(error, match=text):
            append(**bad)
    shifted = torch.zeros(4 * 2 * 8 * 16 + 1, device=device)[1:].view(4, 2, 8, 16)
    for bad, error, text in [
        (dict(q=q[0]), ValueError, "q must be"),
        (dict(q=q[:, :3]), ValueError, "divisor"),
        (dict(q=q.half()), TypeError, "cache's dtype"),
        (dict(q=q[:, :, :8]), ValueError, "expected 2 of"),
        (dict(kc=shifted), ValueError, "aligned"),
        (dict(n=start[:1]), ValueError, "lengths must be"),
        (dict(t=table[0]), ValueError, "page_table must be"),
        (dict(scale=math.inf), ValueError, "scale"),
        (dict(q=q.clone().requires_grad_()), ValueError, "no_grad"),
    ]:
        with pytest.raises(error, match=text):
            attend(**bad)
    small = torch.zeros(4, 2, 8, 12, device=device)
    with pytest.raises(ValueError, match="multiple of 8"):
        attend(q=q[:, :, :12], kc=small, vc=small)
    with pytest.raises(ValueError, match="rotary_dim"):
        ops.rotary_table(4, 3)
    with torch.no_grad():
        assert append(k=k.clone().requires_grad_()) is None
    if device == "cuda":
        with pytest.raises(ValueError, match="is on"):
            attend(n=start.cpu())


@pytest.mark.parametrize("device", DEVICES)
def test_forward_derivatives(device):
    """A direct call's tangent is the gradient's product with it; what has no
    derivative refuses one."""
    fw = torch.autograd.forward_ad
    g = gen(21)
    logits, t = torch.randn(2, 3, 5, 17, generator=g).to(device)
    tokens = torch.randint(0, 17, (3, 5), generator=g).to(device)
    lp, tlp, old, ref = torch.randn(4, 3, 5, generator=g).to(device)
    adv = torch.randn(3, 1, generator=g).to(device)

    def losses(x):
        out = ops.token_policy_loss(x, old, adv, None, ref, kl_coeff=0.1, entropy_coeff=0.2)
        return [*out[:4], out.ess]

    leaf = logits.clone().requires_grad_()
    value = ops.token_log_probs(leaf, tokens)
    want = torch.stack([(torch.autograd.grad(v, leaf, retain_graph=True)[0] * t).sum()
                        for v in value.flatten()]).view(3, 5)
    with fw.dual_level():
        got = fw.unpack_dual(ops.token_log_probs(fw.make_dual(logits, t), tokens))
        assert got.tangent is not None and torch.allclose(got.tangent, want, atol=1e-5)
        assert torch.allclose(got.primal, value, atol=1e-5)
        # a level by itself changes nothing
        assert torch.equal(ops.token_log_probs(logits, tokens), value)
        x = lp.clone().requires_grad_()
        for got, one in zip(losses(fw.make_dual(lp, tlp)), losses(x)):
            (want,) = torch.autograd.grad(one, x, retain_graph=True)
            assert torch.allclose(fw.unpack_dual(got).tangent, (want * tlp).sum(), atol=1e-4)
        k_cache, v_cache = torch.zeros(2, 4, 1, 8, 16, device=device)
        table = torch.zeros(3, 1, dtype=torch.int32, device=device)
        start = torch.zeros(3, dtype=torch.int32, device=device)
        k = torch.zeros(3, 1, 1, 16, device=device)
        dual = fw.make_dual(k, k)
        with pytest.raises(ValueError, match="derivative"), torch.no_grad():
            ops.paged_kv_append(dual, k, k_cache, v_cache, table, start)
        with pytest.raises(ValueError, match="derivative"):
            ops.paged_attention_decode(dual[:, 0], k_cache, v_cache, table, start)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("which", [0, 1])
def test_append_refuses_learned_rotations(device, which):
    """Tables that require a gradient would get none: the GPU's queries carried
    no graph where the CPU's did."""
    k_cache, v_cache = torch.zeros(2, 4, 1, 8, 16, device=device)
    table = torch.zeros(3, 1, dtype=torch.int32, device=device)
    start = torch.zeros(3, dtype=torch.int32, device=device)
    k = torch.zeros(3, 1, 1, 16, device=device)
    rope = list(ops.rotary_table(8, 16, device=device))
    rope[which].requires_grad_()
    with pytest.raises(ValueError, match="rope requires a gradient"):
        ops.paged_kv_append(k, k, k_cache, v_cache, table, start, q=k, rope=tuple(rope))
    with torch.no_grad():
        assert ops.paged_kv_append(k, k, k_cache, v_cache, table, start, q=k, rope=tuple(rope)).shape == k.shape
