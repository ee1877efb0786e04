"""Policy and preference losses on the CPU: the formulas against loops over positions, gradients against differences, hidden
positions, refusals."""
import math

import pytest
import torch

from speech_b200 import ops


def batch(n=4, t=5, c=None, v=11, seed=0, dtype=torch.float64):
    g = torch.Generator().manual_seed(seed)
    shape = (n, t) if c is None else (n, t, c)
    logits = (2 * torch.randn(shape + (v,), generator=g, dtype=torch.float64)).to(dtype)
    targets = torch.randint(0, v, shape, generator=g)
    mask = torch.rand((n, t), generator=g) < 0.7
    mask[0] = True
    mask[1] = False
    near = torch.log_softmax(logits.double(), -1).gather(-1, targets.unsqueeze(-1)).squeeze(-1)
    old = (near + 0.3 * torch.randn(shape, generator=g)).float()
    ref = (near + 0.3 * torch.randn(shape, generator=g)).float()
    adv = torch.randn(n, generator=g)
    return logits, targets, mask, old, ref, adv


def positions(targets, mask):
    for idx in torch.cartesian_prod(*[torch.arange(s) for s in targets.shape]).tolist():
        if bool(mask[idx[0], idx[1]]):
            yield tuple(idx)


def logprob(logits, targets, i):
    x = logits[i].double()
    return float(x[targets[i]] - torch.logsumexp(x, 0))


@pytest.mark.parametrize("c", [None, 3])
@pytest.mark.parametrize("kl", [0.0, 0.07])
def test_policy_loss_formula(c, kl):
    logits, targets, mask, old, ref, adv = batch(c=c)
    loss, logp = ops.policy_loss(logits, targets, mask, old, adv, ref_logp=ref if kl else None, clip=0.1, clip_high=0.25, kl_beta=kl)
    total, count = 0.0, 0
    for i in positions(targets, mask):
        lp, a = logprob(logits, targets, i), float(adv[i[0]])
        assert float(logp[i]) == pytest.approx(lp, rel=2 ** -23)
        r = math.exp(lp - float(old[i]))
        total -= min(r * a, min(max(r, 0.9), 1.25) * a)
        if kl:
            d = float(ref[i]) - lp
            total += kl * (math.exp(d) - d - 1)
        count += 1
    assert float(loss) == pytest.approx(total / count, rel=1e-6)
    hidden = ~mask if c is None else ~mask.unsqueeze(-1).expand(targets.shape)
    assert bool((logp[hidden] == 0).all())


@pytest.mark.parametrize("loss_type", ["dpo", "ipo", "rpo_sq"])
def test_preference_loss_formula(loss_type):
    logits, targets, mask, _, ref, _ = batch(n=6, c=2)
    gap, beta = torch.tensor([0.5, -0.2, 0.1]), 0.3
    loss, rewards = ops.preference_loss(logits, targets, mask, ref, beta=beta, loss_type=loss_type, reward_gap=gap)
    ratio = [0.0] * 6
    for i in positions(targets, mask):
        ratio[i[0]] += logprob(logits, targets, i) - float(ref[i])
    assert rewards.tolist() == pytest.approx([beta * r for r in ratio], rel=1e-6, abs=1e-9)
    want = 0.0
    for n in range(3):
        m = ratio[n] - ratio[n + 3]
        want += {"dpo": math.log1p(math.exp(-beta * m)), "ipo": (m - 0.5 / beta) ** 2, "rpo_sq": (beta * m - float(gap[n])) ** 2}[loss_type] / 3
    assert float(loss) == pytest.approx(want, rel=1e-6)


@pytest.mark.parametrize("what", ["policy", "dpo", "ipo", "rpo_sq"])
def test_gradients_against_differences(what):
    logits, targets, mask, old, ref, adv = batch(n=4, t=3, v=5)

    def f(x):
        if what == "policy":
            return ops.policy_loss(x, targets, mask, old, adv, ref_logp=ref, kl_beta=0.1)[0]
        return ops.preference_loss(x, targets, mask, ref, beta=0.5, loss_type=what, reward_gap=torch.tensor([0.3, 0.1]))[0]

    x = logits.clone().requires_grad_()
    (g,) = torch.autograd.grad(f(x), x)
    # losses come out in fp32 (values up to 2^3: steps of 2^-20 halved): a central difference over 2h = 1/16 is off by up to 2^-20 / 2^-4
    # = 2^-16 from rounding and h^2 / 6 |f'''| (h = 2^-5, third derivatives of these losses below 8) = 1.3e-3 from curvature
    h = 2.0 ** -5
    for i in torch.cartesian_prod(*[torch.arange(s) for s in logits.shape]).tolist():
        d = torch.zeros_like(logits)
        d[tuple(i)] = h
        slope = (float(f(logits + d)) - float(f(logits - d))) / (2 * h)
        near_clip = what == "policy" and min(abs(math.exp(logprob(logits, targets, tuple(i[:-1])) - float(old[tuple(i[:-1])])) - b) for b in (0.8, 1.2)) < 0.1
        if not near_clip:                                   # the clipped term has a corner there
            assert float(g[tuple(i)]) == pytest.approx(slope, abs=1.4e-3)


def test_hidden_positions_have_no_influence_and_empty_batches_give_zero():
    logits, targets, mask, old, ref, adv = batch()
    bad = logits.clone()
    bad[~mask] = float("nan")
    bad_t = targets.masked_fill(~mask, -100)
    for x, t in ((logits, targets), (bad, bad_t)):
        x.requires_grad_()
    a, b = (ops.policy_loss(x, t, mask, old, adv, ref_logp=ref, kl_beta=0.1) for x, t in ((logits, targets), (bad, bad_t)))
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    ga, gb = torch.autograd.grad(a[0], logits)[0], torch.autograd.grad(b[0], bad)[0]
    assert torch.equal(ga, gb) and bool((gb[~mask] == 0).all())
    loss, _ = ops.policy_loss(logits, targets, torch.zeros_like(mask), old, adv)
    assert float(loss) == 0.0
    loss, rewards = ops.preference_loss(logits, targets, torch.zeros_like(mask), ref)
    assert float(loss) == pytest.approx(math.log(2)) and bool((rewards == 0).all())
    loss, logp = ops.policy_loss(logits[:, :0], targets[:, :0], mask[:, :0], old[:, :0], adv)
    assert float(loss) == 0.0 and logp.shape == (4, 0)


def test_gradients_go_to_the_logits_only():
    """Log-probabilities, advantages and gaps that require gradients: the loss does not on their account, and they get none."""
    logits, targets, mask, old, ref, adv = batch()
    gap = torch.rand(2).requires_grad_()
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


def test_refusals():
    logits, targets, mask, old, ref, adv = batch()
    with pytest.raises(ValueError, match="ref_logp"):
        ops.policy_loss(logits, targets, mask, old, adv, kl_beta=0.1)
    with pytest.raises(ValueError, match="clip"):
        ops.policy_loss(logits, targets, mask, old, adv, clip=-0.1)
    with pytest.raises(ValueError, match="targets"):
        ops.policy_loss(logits, targets[:, :-1], mask, old, adv)
    with pytest.raises(ValueError, match="targets"):
        ops.policy_loss(logits, targets.float(), mask, old, adv)
    with pytest.raises(ValueError, match="mask"):
        ops.policy_loss(logits, targets, mask[:, :-1], old, adv)
    with pytest.raises(ValueError, match="old_logp"):
        ops.policy_loss(logits, targets, mask, old[:-1], adv)
    with pytest.raises(ValueError, match="advantages"):
        ops.policy_loss(logits, targets, mask, old, adv[:-1])
    with pytest.raises(ValueError, match="logits"):
        ops.policy_loss(logits[0], targets[0], mask[0], old[0], adv)
    with pytest.raises(ValueError, match="pairs"):
        ops.preference_loss(logits[:3], targets[:3], mask[:3], ref[:3])
    with pytest.raises(ValueError, match="reward gap"):
        ops.preference_loss(logits, targets, mask, ref, loss_type="rpo_sq")
    with pytest.raises(ValueError, match="reward_gap"):
        ops.preference_loss(logits, targets, mask, ref, loss_type="rpo_sq", reward_gap=torch.zeros(4))
    with pytest.raises(NotImplementedError):
        ops.preference_loss(logits, targets, mask, ref, loss_type="hinge")


def test_refusals_of_scalars():
    _, targets, mask, old, ref, adv = batch()
    none = torch.zeros(())
    with pytest.raises(ValueError, match="logits"):
        ops.policy_loss(none, targets, mask, old, adv)
    with pytest.raises(ValueError, match="logits"):
        ops.preference_loss(none, targets, mask, ref)
    logits = batch()[0]
    with pytest.raises(ValueError, match="beta"):
        ops.preference_loss(logits, targets, mask, ref, beta=0.0, loss_type="ipo")
