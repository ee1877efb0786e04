"""Policy and preference loss kernels against a plain statement in 64 bits."""
import pytest
import torch

pytestmark = pytest.mark.gpu

EPS = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}      # half a step, relative


def make(n, t, c, v, dtype, seed=0, scale=2.0, whole=False):
    g = torch.Generator(device="cuda").manual_seed(seed)
    shape = (n, t) if c is None else (n, t, c)
    logits = (scale * torch.randn(shape + (v,), generator=g, device="cuda")).to(dtype)
    targets = torch.randint(0, v, shape, generator=g, device="cuda")
    mask = torch.rand((n, t), generator=g, device="cuda") < 0.7
    mask[0, 0] = True
    if n > 2:
        mask[2] = False
    if whole:
        mask[:] = True
    near = torch.log_softmax(logits.double(), -1).gather(-1, targets.unsqueeze(-1)).squeeze(-1)
    old = (near + 0.2 * torch.randn(shape, generator=g, device="cuda")).float()
    ref = (near + 0.2 * torch.randn(shape, generator=g, device="cuda")).float()
    adv = torch.randn(n, generator=g, device="cuda")
    return logits, targets, mask, old, ref, adv


def plain_logp(logits, targets, mask):
    m = mask.view(mask.shape + (1,) * (targets.dim() - 2)).expand(targets.shape)
    x = logits.double().masked_fill(~m.unsqueeze(-1), 0.0)
    lse = torch.logsumexp(x, -1)
    lp = (x.gather(-1, targets.masked_fill(~m, 0).unsqueeze(-1)).squeeze(-1) - lse) * m
    return lp, m, torch.exp(x - lse.unsqueeze(-1))


def lp_tolerance(v):
    # CUDA states 2 + floor(1.173 |x|) ulp (2^-23) for the fast exponential; weighted by the exponentials themselves, |x| averages to
    # the distance from the largest logit, below 16 here: 21 * 2^-23 < 2^-18.  A thread adds up to max(64, v / 512) terms one by one,
    # half a step each.  fp32 storage of a logp below 32 adds 2^-20.
    return 2.0 ** -18 + max(64, v // 512 + 16) * 2.0 ** -24 + 2.0 ** -20


def check_gradient(got, targets, weights, slope, dtype, v, upstream=1.0):
    """slope: 64-bit dloss/dlogp per position (times the upstream gradient)."""
    want = -weights * slope.unsqueeze(-1)
    want.scatter_add_(-1, targets.clamp(0, v - 1).unsqueeze(-1), slope.unsqueeze(-1))
    # one rounding of the result; softmax weights inherit the log-probability's error and one more exponential; the slope is fp32
    # and for the policy loss its ratio inherits the log-probability's error as well
    lp = 2 * lp_tolerance(v) + 2.0 ** -18
    tol = EPS[dtype] * want.abs() + slope.abs().unsqueeze(-1) * (weights + (want.abs() > 0)) * 2 * lp + 2.0 ** -25 * (dtype == torch.float16) + 1e-38
    assert bool(((got.double() - want).abs() <= tol).all()), float(((got.double() - want).abs() / tol).max())


SHAPES = [(2, 3, None, 2), (4, 5, 8, 130), (3, 4, None, 257), (4, 6, 8, 2024), (2, 3, 2, 2049), (2, 5, None, 16384), (2, 3, None, 20003), (2, 2, None, 151936), (1, 1, 1, 1)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("kl", [0.0, 0.04])
def test_policy_loss(shape, dtype, kl):
    from speech_b200 import ops

    n, t, c, v = shape
    logits, targets, mask, old, ref, adv = make(n, t, c, v, dtype)
    up = 512.0 if dtype == torch.float16 else 1.0
    lp, m, w = plain_logp(logits, targets, mask)
    for border in (0.8, 1.3):                                # no input lies on a clip border, where the slope jumps
        old = torch.where((torch.exp(lp - old.double()) - border).abs() < 1e-3, old + 0.01, old)
    x = logits.clone().requires_grad_()
    loss, logp = ops.policy_loss(x, targets, mask, old, adv, ref_logp=ref if kl else None, clip=0.2, clip_high=0.3, kl_beta=kl)
    (g,) = torch.autograd.grad(loss, x, torch.tensor(up, device="cuda"))
    tol = lp_tolerance(v)
    assert bool(((logp.double() - lp).abs() <= tol + EPS[torch.float32] * lp.abs()).all())
    assert bool((logp[~m] == 0).all())
    a = adv.double().view((-1,) + (1,) * (targets.dim() - 1))
    r = torch.exp(lp - old.double())
    plain, clipped = r * a, r.clamp(0.8, 1.3) * a
    term, slope = -torch.minimum(plain, clipped), torch.where(plain <= clipped, -plain, 0.0)
    if kl:
        d = ref.double() - lp
        term, slope = term + kl * (torch.exp(d) - d - 1), slope + kl * (1 - torch.exp(d))
    count = m.sum().clamp(min=1)
    want = (term * m).sum() / count
    reach = (((r * a).abs() + kl * (1 + torch.exp(ref.double() - lp))) * m).sum() / count          # how far the loss moves with the log-probabilities
    assert abs(float(loss) - float(want)) <= 2.0 ** -23 * abs(float(want)) + float(reach) * tol
    # the slope itself moves with the log-probability: r a and kl exp(d) by the same relative error
    check_gradient(g, targets, w, slope * m / count * up, dtype, v)
    hidden = ~m
    assert bool((g[hidden] == 0).all())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("shape", SHAPES[:-1])
@pytest.mark.parametrize("kind", ["dpo", "ipo", "rpo_sq"])
def test_preference_loss(shape, dtype, kind):
    from speech_b200 import ops

    n, t, c, v = shape
    n += n % 2
    logits, targets, mask, _, ref, _ = make(n, t, c, v, dtype, seed=1)
    beta, up, pairs = 0.1, 64.0 if dtype == torch.float16 else 1.0, n // 2
    gap = torch.rand(pairs, device="cuda", generator=torch.Generator(device="cuda").manual_seed(3))
    x = logits.clone().requires_grad_()
    loss, rewards = ops.preference_loss(x, targets, mask, ref, beta=beta, loss_type=kind, reward_gap=gap)
    (g,) = torch.autograd.grad(loss, x, torch.tensor(up, device="cuda"))
    lp, m, w = plain_logp(logits, targets, mask)
    ratio = ((lp - ref.double()) * m).flatten(1).sum(1)
    margin = ratio[:pairs] - ratio[pairs:]
    tol = lp_tolerance(v) * m.flatten(1).sum(1).max()                                           # positions of a sequence, all off the same way
    if kind == "dpo":
        each, slope, bend = -torch.nn.functional.logsigmoid(beta * margin), -beta * torch.sigmoid(-beta * margin), beta ** 2
    elif kind == "ipo":
        each, slope, bend = (margin - 0.5 / beta) ** 2, 2 * (margin - 0.5 / beta), 2.0
    else:
        each, slope, bend = (beta * margin - gap.double()) ** 2, 2 * beta * (beta * margin - gap.double()), 2 * beta ** 2
    assert bool(((rewards.double() - beta * ratio).abs() <= beta * tol + 2.0 ** -23 * (beta * ratio).abs()).all())
    assert abs(float(loss) - float(each.mean())) <= float(slope.abs().max() * 2 * tol + bend * (2 * tol) ** 2) + 2.0 ** -23 * float(each.mean())
    s = torch.cat([slope, -slope]).view((-1,) + (1,) * (targets.dim() - 1)) * m / pairs * up
    want = -w * s.unsqueeze(-1)
    want.scatter_add_(-1, targets.unsqueeze(-1), s.unsqueeze(-1))
    one = lp_tolerance(v) * 2 + 2.0 ** -17
    allow = EPS[dtype] * want.abs() + (s.abs() * one + m * bend * 2 * tol / pairs * up).unsqueeze(-1) * (w + torch.zeros_like(w).scatter_(-1, targets.unsqueeze(-1), 1.0)) \
        + 2.0 ** -25 * (dtype == torch.float16) + 1e-38
    assert bool(((g.double() - want).abs() <= allow).all()), float(((g.double() - want).abs() / allow).max())


def test_strided_logits_and_hidden_garbage():
    """Logits that are a slice of a longer tensor (rows at odd addresses), NaN and invalid targets at hidden positions."""
    from speech_b200 import ops

    logits, targets, mask, old, ref, adv = make(4, 7, 3, 333, torch.bfloat16)
    longer = torch.full((4, 9, 3, 335), float("nan"), dtype=torch.bfloat16, device="cuda")
    view = longer[:, 1:8, :, 1:334]
    view.copy_(logits)
    view[~mask] = float("nan")
    t = targets.masked_fill(~mask.unsqueeze(-1), -100)

    def policy(x, y):
        return ops.policy_loss(x, y, mask, old, adv, ref_logp=ref, kl_beta=0.1)

    for f in (policy, lambda x, y: ops.preference_loss(x, y, mask, ref)):
        a, b = logits.clone().requires_grad_(), view.detach().requires_grad_()
        (la, ea), (lb, eb) = f(a, targets), f(b, t)
        # a row's groups start at another address, so its sum is taken in another order: both sides are within the log-probability's
        # tolerance of the same value (times the 21 positions of a sequence for the rewards of the second loss, beta = 0.1)
        assert bool(((ea.double() - eb.double()).abs() <= 2 * lp_tolerance(333) * (1 if f is policy else 2.1)).all())
        assert bool((la.double() - lb.double()).abs() <= 2 * lp_tolerance(333) * 2.1 + 2.0 ** -23 * la.double().abs())
        ga, gb = torch.autograd.grad(la, a)[0], torch.autograd.grad(lb, b)[0]
        # and one step of the gradient's type
        assert bool(((ga.double() - gb.double()).abs() <= 2.0 ** -7 * ga.double().abs() + 1e-12).all())


def test_second_backward_other_upstream_and_determinism():
    from speech_b200 import ops

    logits, targets, mask, old, ref, adv = make(8, 33, 8, 2024, torch.bfloat16)
    x = logits.clone().requires_grad_()

    def f():
        return ops.policy_loss(x, targets, mask, old, adv, ref_logp=ref, kl_beta=0.04)[0]

    loss = f()
    (a,) = torch.autograd.grad(loss, x, retain_graph=True)
    kept = a.clone()
    (b,) = torch.autograd.grad(loss, x, torch.tensor(0.5, device="cuda"), retain_graph=True)
    assert torch.equal(a, kept), "a second backward pass has written into the first one's gradient"
    (c,) = torch.autograd.grad(loss, x)
    again = f()
    (d,) = torch.autograd.grad(again, x)
    assert torch.equal(loss, again) and torch.equal(a, d)
    # recomputed from memory: another exponential, one step of the result's type apart at most
    assert bool(((c.double() - a.double()).abs() <= 2.0 ** -7 * a.double().abs() + 1e-12).all())
    assert bool(((2 * b.double() - a.double()).abs() <= 2.0 ** -7 * a.double().abs() + 1e-12).all())
    p = ops.preference_loss(x, targets, mask, ref)[0]
    assert torch.equal(torch.autograd.grad(p, x, retain_graph=True)[0], torch.autograd.grad(p, x)[0])


def test_invalid_target_is_loud_and_stays_in_bounds():
    from speech_b200 import ops

    logits, targets, mask, old, ref, adv = make(2, 3, None, 64, torch.bfloat16, whole=True)
    for bad in (-1, 64, 2 ** 40):
        t = targets.clone()
        t[0, 1] = bad
        loss, logp = ops.policy_loss(logits, t, mask, old, adv)
        assert bool(torch.isnan(loss)) and bool(torch.isnan(logp[0, 1])) and not bool(torch.isnan(logp[1]).any())


def test_extreme_logits():
    """The type's lowest value and -inf as vocabulary masks, a row that is all one value."""
    from speech_b200 import ops

    logits, targets, mask, old, ref, adv = make(2, 4, None, 500, torch.bfloat16, whole=True)
    targets.clamp_(max=249)
    logits[0, :, 250:] = float("-inf")
    logits[1, :, 250:] = torch.finfo(torch.bfloat16).min
    logits[1, 3] = 3.0
    x = logits.clone().requires_grad_()
    loss, logp = ops.policy_loss(x, targets, mask, old, adv, ref_logp=ref, kl_beta=0.1)
    (g,) = torch.autograd.grad(loss, x)
    assert bool(torch.isfinite(loss)) and bool(torch.isfinite(g).all())
    assert bool((g[0, :, 250:] == 0).all()) and bool((g[1, :3, 250:] == 0).all())
    lp, _, _ = plain_logp(logits, targets, mask)
    assert bool(((logp.double() - lp).abs() <= lp_tolerance(500)).all())
    # a row of nothing but the lowest value is uniform: weights of 1 / 500, in the gradient that forward writes and in the one read again
    x = logits.clone()
    x[1, 2] = torch.finfo(torch.bfloat16).min
    x.requires_grad_()
    loss, logp = ops.policy_loss(x, targets, mask, old, adv)
    (g,) = torch.autograd.grad(loss, x, retain_graph=True)
    (h,) = torch.autograd.grad(loss, x)
    r = torch.exp(-torch.log(torch.tensor(500.0, dtype=torch.float64, device="cuda")) - old[1, 2].double())
    slope = -float(r) * float(adv[1]) / mask.sum().item() if not (float(adv[1]) > 0 and float(r) > 1.2 or float(adv[1]) < 0 and float(r) < 0.8) else 0.0
    for got in (g, h):
        want = torch.full((500,), -slope / 500, dtype=torch.float64, device="cuda")
        want[targets[1, 2]] += slope
        assert bool(((got[1, 2].double() - want).abs() <= 2.0 ** -8 * want.abs() + abs(slope) * 2.0 ** -15).all())
    p, _ = ops.preference_loss(x, targets, mask, old)
    assert bool(torch.isfinite(torch.autograd.grad(p, x)[0]).all())


def test_forward_mode_derivatives_are_refused():
    import torch.autograd.forward_ad as forward_ad

    from speech_b200 import ops

    logits, targets, mask, old, ref, adv = make(2, 3, None, 64, torch.bfloat16)
    with forward_ad.dual_level():
        x = forward_ad.make_dual(logits, torch.ones_like(logits))
        with pytest.raises(NotImplementedError):
            ops.policy_loss(x, targets, mask, old, adv)
        with pytest.raises(NotImplementedError):
            ops.preference_loss(x, targets, mask, ref)


def test_gradients_go_to_the_logits_only():
    """Log-probabilities, advantages and gaps that require gradients: the loss does not on their account, and they get none."""
    from speech_b200 import ops

    logits, targets, mask, old, ref, adv = make(4, 3, None, 64, torch.bfloat16)
    gap = torch.rand(2, device="cuda").requires_grad_()
    for t in (old, ref, adv):
        t.requires_grad_()
    losses = (lambda x: ops.policy_loss(x, targets, mask, old, adv, ref_logp=ref, kl_beta=0.1)[0],
              lambda x: ops.preference_loss(x, targets, mask, ref, loss_type="rpo_sq", reward_gap=gap)[0])
    for f in losses:
        assert not f(logits.detach()).requires_grad
        x = logits.detach().clone().requires_grad_()
        f(x).backward()
        assert x.grad is not None and float(x.grad.abs().max()) > 0
    assert all(t.grad is None for t in (old, ref, adv, gap))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_kl_term_near_the_reference(dtype):
    """exp(d) - d - 1 of log ratios down to 1e-5.  Rows of equal logits, 2^k of them: their log-probability is -k ln 2 to the last of 64 bits, so
    that the term's own error shows."""
    import math

    from speech_b200 import ops

    for k in (1, 7, 11, 16):
        logits = torch.full((1, 40, 2 ** k), -3.0, device="cuda").to(dtype)
        targets, none = torch.zeros((1, 40), dtype=torch.long, device="cuda"), torch.zeros(1, device="cuda")
        lp = -k * math.log(2.0)
        for size in (1e-5, 1e-4, 1e-3, 0.01, 0.1, 0.499, 0.501, 2.0):
            for sign in (-1.0, 1.0):
                ref = torch.linspace(size / 2, size, 40, dtype=torch.float64, device="cuda").mul(sign).add(lp).float().view(1, 40)
                d = ref.double() - lp
                # 64-bit term by the series where the difference would cancel there, too (the rest of six terms is below 1e-13 of it)
                want = torch.where(d.abs() < 0.02, d * d * (1 / 2 + d * (1 / 6 + d * (1 / 24 + d * (1 / 120 + d * (1 / 720 + d / 5040))))), torch.expm1(d) - d)
                loss, logp = ops.policy_loss(logits, targets, None, logp_of(lp, ref), none, ref_logp=ref, kl_beta=1.0)
                # d to half a step, twice in d^2; nine operations; above 1/2 the library's expm1 and d, two units at most, in a difference of at
                # least a seventh of them (expm1(d) / (expm1(d) - d) = 4.4 at 1/2, 3.7 at -1/2)
                assert abs(float(loss) / float(want.mean()) - 1) <= 16 * 2.0 ** -24 * (1 if size < 0.5 else 3), (k, size, sign)


def logp_of(lp, like):
    return torch.full_like(like, lp)


def test_what_backward_needs_is_seen_by_autograd():
    """The gradient that the forward pass writes, and the rows' statistics, go through saved variables."""
    from torch.utils.checkpoint import checkpoint

    from speech_b200 import ops

    logits, targets, mask, old, ref, adv = make(8, 64, None, 2024, torch.bfloat16)
    size = logits.numel() * logits.element_size()
    for f in (lambda x: ops.policy_loss(x, targets, mask, old, adv, ref_logp=ref, kl_beta=0.04)[0], lambda x: ops.preference_loss(x, targets, mask, ref)[0]):
        x = logits.detach().clone().requires_grad_()
        loss = f(x)
        (want,) = torch.autograd.grad(loss, x)
        with torch.autograd.graph.save_on_cpu():
            before = torch.cuda.memory_allocated()
            loss = f(x)
            assert torch.cuda.memory_allocated() - before < size // 8
        assert torch.equal(torch.autograd.grad(loss, x)[0], want)
        loss = checkpoint(f, x, use_reentrant=False)
        assert torch.equal(torch.autograd.grad(loss, x)[0], want)
        # a gradient that its owner changes does not reach a further backward pass
        loss = f(x)
        (g,) = torch.autograd.grad(loss, x, retain_graph=True)
        g.zero_()
        (h,) = torch.autograd.grad(loss, x)
        # computed from memory: another exponential, a step of the type apart at most
        assert bool(((h.double() - want.double()).abs() <= 2.0 ** -7 * want.double().abs() + 1e-12).all())


def test_captured_and_replayed():
    from speech_b200 import ops

    logits, targets, mask, old, ref, adv = make(4, 9, 2, 2024, torch.bfloat16)
    x = logits.clone().requires_grad_()

    def step():
        loss, logp = ops.policy_loss(x, targets, mask, old, adv, ref_logp=ref, kl_beta=0.04)
        (g,) = torch.autograd.grad(loss, x)
        p, rewards = ops.preference_loss(x, targets, mask, ref)
        (h,) = torch.autograd.grad(p, x)
        return loss, logp, g, p, rewards, h

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    other = make(4, 9, 2, 2024, torch.bfloat16, seed=9)
    with torch.no_grad():
        x.copy_(other[0])
    for a, b in zip((targets, mask, old, ref, adv), other[1:]):
        a.copy_(b)
    graph.replay()
    want = [o.detach().clone() for o in step()]
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(out, want))


@pytest.mark.parametrize("v", [130, 2024, 9000, 40001])
def test_infinite_and_nan_logits(v):
    """-inf logits (a masked vocabulary) have no weight and no gradient; a NaN or +inf logit shows in the loss and its sequence's reward."""
    from speech_b200 import ops

    logits, targets, mask, old, ref, adv = make(4, 5, None, v, torch.bfloat16)
    mask[:] = True
    hide = torch.rand(logits.shape, device="cuda", generator=torch.Generator(device="cuda").manual_seed(3)) < 0.5
    hide[..., : v // 3] = True
    hide.scatter_(-1, targets.unsqueeze(-1), False)
    logits = logits.masked_fill(hide, float("-inf"))
    lp, m, weights = plain_logp(logits, targets, mask)
    old, tol = lp.float(), lp_tolerance(v)
    x = logits.clone().requires_grad_()
    loss, logp = ops.policy_loss(x, targets, mask, old, adv)
    assert bool(((logp.double() - lp).abs() <= tol).all())
    # the old log-probabilities are the new ones (to fp32): r = 1, the slope -A / count
    g, slope = torch.autograd.grad(loss, x)[0], -adv.double().view(-1, 1) / m.sum()
    check_gradient(g, targets, weights, slope.expand(targets.shape), torch.bfloat16, v)
    assert bool((g[hide] == 0).all())
    loss, rewards = ops.preference_loss(x, targets, mask, old)
    # every position within the tolerance of its log-probability, and old's rounding (2^-20 below 32) on top
    assert bool((rewards.double().abs() <= 0.1 * 5 * (tol + 2.0 ** -20)).all())
    h = torch.autograd.grad(loss, x)[0]
    assert bool((h[hide] == 0).all()) and bool(torch.isfinite(h).all())
    for bad in (float("nan"), float("inf")):
        for at in (0, v // 2, v - 1):
            y = logits.clone()
            y[1, 2, at] = bad
            y.requires_grad_()
            a, logp = ops.policy_loss(y, targets, mask, old, adv)
            b, rewards = ops.preference_loss(y, targets, mask, old)
            assert bool(torch.isnan(a)) and bool(torch.isnan(b)) and bool(torch.isnan(logp[1, 2])) and int(torch.isnan(logp).sum()) == 1
            assert bool(torch.isnan(rewards[1])) and int(torch.isnan(rewards).sum()) == 1


def far_logits(how, v, dtype):
    """Logits far below zero, [4, 134, v]: every row shifted by another amount in [-300, -60], the first ids or a whole row at the type's lowest value."""
    logits, targets, mask, _, _, adv = make(4, 134, None, v, torch.float32, seed=v, whole=True)
    low = torch.finfo(dtype).min
    if how == "shifted":
        logits = logits - torch.linspace(60.0, 300.0, 4 * 134, device="cuda").view(4, 134, 1)
    elif how == "first ids lowest":
        n = min(10000, v // 2)
        logits[..., :n] = low
        targets = n + targets % (v - n)
    else:
        logits[0] = low
        logits[1] = -88.7
        logits[2, :, ::2] = low
        logits[2, :, 1::2] = -266.0
        targets[2] = targets[2] // 2 * 2 + 1 - 2 * (targets[2] // 2 * 2 + 1 >= v).long()
    logits = logits.to(dtype)
    # relative to the maximum first: the lowest value plus the logarithm of the row's size is the lowest value, in 64 bits too
    lp, m, w = plain_logp(logits.double() - logits.double().amax(-1, keepdim=True), targets, mask)
    g = torch.Generator(device="cuda").manual_seed(1)
    # ratios 0.5 to 2 that are not on a border of the clip range
    apart = torch.tensor([-0.7, -0.3, -0.1, 0.1, 0.25, 0.7], device="cuda")[torch.randint(0, 6, lp.shape, generator=g, device="cuda")]
    old, ref = (lp - apart).float(), (lp + 0.2 * torch.randn(lp.shape, generator=g, device="cuda")).float()
    return logits, targets, mask, old, ref, adv, lp, m, w


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("v", [130, 500, 2024, 9000, 40001])
@pytest.mark.parametrize("how", ["shifted", "first ids lowest", "whole rows"])
def test_logits_far_below_zero(how, v, dtype):
    """A thread's share of a row that is still empty when it meets a maximum far below zero adds nothing, in both losses."""
    from speech_b200 import ops

    logits, targets, mask, old, ref, adv, lp, m, w = far_logits(how, v, dtype)
    tol, up = lp_tolerance(v), 512.0 if dtype == torch.float16 else 1.0
    x = logits.clone().requires_grad_()
    loss, logp = ops.policy_loss(x, targets, mask, old, adv, ref_logp=ref, kl_beta=0.04)
    (g,) = torch.autograd.grad(loss, x, torch.tensor(up, device="cuda"))
    assert bool(((logp.double() - lp).abs() <= tol + EPS[torch.float32] * lp.abs()).all())
    a, r, d = adv.double().view(-1, 1), torch.exp(lp - old.double()), ref.double() - lp
    plain, clipped = r * a, r.clamp(0.8, 1.2) * a
    term, slope = -torch.minimum(plain, clipped) + 0.04 * (torch.exp(d) - d - 1), torch.where(plain <= clipped, -plain, 0.0) + 0.04 * (1 - torch.exp(d))
    reach = ((r * a).abs() + 0.04 * (1 + torch.exp(d))).mean()                                    # how far the loss moves with the log-probabilities
    assert abs(float(loss) - float(term.mean())) <= 2.0 ** -23 * abs(float(term.mean())) + float(reach) * tol
    # as check_gradient, but the slope's two parts may cancel: each moves with the log-probability by its own size (d/dlp of r a and of
    # 0.04 (1 - exp(d))), which is no longer within the log-probability's error of their sum
    s = (slope / lp.numel() * up).unsqueeze(-1)
    moves = (torch.where(plain <= clipped, plain.abs(), 0.0) + 0.04 * (1 + torch.exp(d))).unsqueeze(-1) / lp.numel() * up * (tol + 2.0 ** -22)
    spread = w + torch.zeros_like(w).scatter_(-1, targets.unsqueeze(-1), 1.0)
    want = -w * s
    want.scatter_add_(-1, targets.unsqueeze(-1), s)
    allow = EPS[dtype] * want.abs() + (s.abs() * 2 * (2 * tol + 2.0 ** -18) + moves) * spread + 2.0 ** -25 * (dtype == torch.float16) + 1e-38
    bad = ((g.double() - want).abs() / allow).max()
    assert float(bad) <= 1.0, float(bad)
    x = logits.clone().requires_grad_()
    loss, rewards = ops.preference_loss(x, targets, mask, ref)
    (g,) = torch.autograd.grad(loss, x, torch.tensor(up, device="cuda"))
    ratio = (lp - ref.double()).sum(1)
    margin = 0.1 * (ratio[:2] - ratio[2:])
    assert bool(((rewards.double() - 0.1 * ratio).abs() <= 13.4 * tol + 2.0 ** -23 * (0.1 * ratio).abs()).all())
    each = -torch.nn.functional.logsigmoid(margin)
    assert abs(float(loss) - float(each.mean())) <= 2 * 13.4 * tol + 2.0 ** -23 * float(each.mean())
    # the slope moves with the margin: by at most 0.1 times the margin's error, relative to the slope's own bound of 0.1 / 2
    s = (0.05 * torch.cat([-torch.sigmoid(-margin), torch.sigmoid(-margin)]) * up).view(-1, 1).expand(lp.shape)
    want = -w * s.unsqueeze(-1)
    want.scatter_add_(-1, targets.unsqueeze(-1), s.unsqueeze(-1))
    allow = EPS[dtype] * want.abs() + (s.abs() * (2 * tol + 2.0 ** -17) + 0.05 * up * 2 * 13.4 * tol).unsqueeze(-1) * spread + 2.0 ** -25 * (dtype == torch.float16) + 1e-38
    bad = ((g.double() - want).abs() / allow).max()
    assert float(bad) <= 1.0, float(bad)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("t,v", [(4096, 2024), (512, 40001), (8192, 200)])
def test_rewards_of_long_sequences_have_no_bias(t, v, dtype):
    """Every row's log sum moves the reward of its sequence, so the exponentials may be off to both sides but not to one."""
    from speech_b200 import ops

    logits, targets, mask, _, _, _ = make(2, t, None, v, dtype, seed=4, whole=True)
    lp, _, w = plain_logp(logits, targets, mask)
    ref = lp.float()
    _, rewards = ops.preference_loss(logits, targets, mask, ref, beta=1.0)
    ratio = (lp - ref.double()).sum(1)
    # an exponential is off by 0.6 units in the last place (2^-23) and its sum with three others by two half steps, at random: at most 1.9e-7
    # of the term, a standard deviation below 1.1e-7; terms of a row weigh w, rows add up; six deviations, and 4e-10 a row to one side
    deviation = 1.1e-7 * (w * w).sum((1, 2)).sqrt()
    if dtype == torch.bfloat16:
        # an exponential's error is a function of its argument, and of the differences of bf16 values there are few: equal ones have equal
        # errors, at most 0.6 * 2^-23 of the term, a deviation of 0.6 * 2^-23 / sqrt(3) for each of them, weighted by all the terms that have it
        x = logits.double()
        same = []
        for i in range(2):
            _, at = torch.unique(x[i] - x[i].amax(-1, keepdim=True), return_inverse=True)
            same.append((torch.zeros(int(at.max()) + 1, dtype=torch.float64, device="cuda").scatter_add_(0, at.flatten(), w[i].flatten()) ** 2).sum().sqrt())
        deviation = deviation + 0.6 * 2.0 ** -23 / 3 ** 0.5 * torch.stack(same)
    bound = t * 4e-10 + 6 * deviation
    assert bool(((rewards.double() - ratio).abs() <= bound + 2.0 ** -24 * ratio.abs()).all()), ((rewards.double() - ratio) / t).tolist()
    # what it tells apart: an exponential that is off by 7e-8 to one side, and from fp32 logits one by 1e-8
    assert float(bound.max()) < t * (1e-8 if dtype == torch.float32 else 7e-8), float(bound.max()) / t


def test_rows_beyond_32_bit_offsets():
    from speech_b200 import ops

    logits, targets, mask, old, ref, adv = make(2, 3, None, 300, torch.bfloat16)
    far = torch.empty(2 ** 31 + 4096, dtype=torch.bfloat16, device="cuda").as_strided((2, 3, 300), (2 ** 31 + 1024, 300, 1))
    far.copy_(logits)
    results = []
    for t in (logits, far):
        x = t.detach().requires_grad_()
        loss, logp = ops.policy_loss(x, targets, mask, old, adv, ref_logp=ref, kl_beta=0.04)
        p, rewards = ops.preference_loss(x, targets, mask, ref)
        results.append([loss, logp, rewards, torch.autograd.grad(loss, x, retain_graph=True)[0], torch.autograd.grad(loss, x)[0], torch.autograd.grad(p, x)[0]])
    assert all(torch.equal(a, b) for a, b in zip(*results))


def test_calls_from_two_threads():
    import threading

    from speech_b200 import ops

    cases, results = [make(4, 50, 2, v, torch.bfloat16, seed=v) for v in (2024, 300)], [[], []]

    def call(c):
        logits, targets, mask, old, ref, adv = c
        x = logits.detach().requires_grad_()
        loss, _ = ops.policy_loss(x, targets, mask, old, adv, ref_logp=ref, kl_beta=0.04)
        p, _ = ops.preference_loss(x, targets, mask, ref)
        return torch.autograd.grad(loss, x)[0], torch.autograd.grad(p, x)[0]

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(10):
                results[i].append(call(cases[i]))
            torch.cuda.current_stream().synchronize()

    torch.cuda.synchronize()
    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for c, got in zip(cases, results):
        want = call(c)
        assert len(got) == 10 and all(torch.equal(a, b) for r in got for a, b in zip(r, want))
