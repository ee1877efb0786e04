"""Cross attention and shared-prefix attention on the CPU: loops over single queries, gradients against differences, hidden places,
refusals."""
import math

import pytest
import torch

from speech_b200 import ops


def one_query(q, keys, values, scale):
    """64-bit attention of one query vector over a list of key / value vectors."""
    if len(keys) == 0:
        return torch.zeros_like(q, dtype=torch.float64)
    s = torch.stack([(q.double() * k.double()).sum() * scale for k in keys])
    w = torch.exp(s - s.max())
    w = w / w.sum()
    return sum(wi * v.double() for wi, v in zip(w, values))


@pytest.mark.parametrize("heads,kv_heads,group", [(2, 2, 1), (4, 2, 1), (4, 1, 3)])
@pytest.mark.parametrize("hide", ["none", "lengths", "mask", "both"])
def test_cross_attention_against_single_queries(heads, kv_heads, group, hide):
    g = torch.Generator().manual_seed(0)
    M, Tq, Tk, D = 3, 2, 5, 8
    q = torch.randn(M * group, Tq, heads, D, generator=g)
    k, v = torch.randn(M, Tk, kv_heads, D, generator=g), torch.randn(M, Tk, kv_heads, D, generator=g)
    lengths = torch.tensor([5, 0, 9]) if hide in ("lengths", "both") else None
    mask = torch.rand(M, Tk, generator=g) < 0.4 if hide in ("mask", "both") else None
    out = ops.cross_attention(q, k, v, key_lengths=lengths, key_mask=mask, scale=0.3)
    assert out.shape == (M * group, Tq, heads * D)
    for b in range(M * group):
        m = b // group
        seen = [j for j in range(Tk) if (lengths is None or j < int(lengths[m])) and (mask is None or not bool(mask[m, j]))]
        for t in range(Tq):
            for h in range(heads):
                hk = h // (heads // kv_heads)
                want = one_query(q[b, t, h], [k[m, j, hk] for j in seen], [v[m, j, hk] for j in seen], 0.3)
                # fp32: a few dozen roundings of 2^-24 on values of order one
                assert torch.allclose(out[b, t, h * D:(h + 1) * D].double(), want, rtol=0, atol=64 * 2.0 ** -24)


def test_gradients_against_differences_and_hidden_garbage():
    g = torch.Generator().manual_seed(1)
    q, k, v = torch.randn(4, 3, 4, 8, generator=g), torch.randn(2, 6, 2, 8, generator=g), torch.randn(2, 6, 2, 8, generator=g)
    mask = torch.tensor([[False, True, False, False, True, False], [True] * 6])
    k[mask], v[mask] = float("nan"), float("inf")
    for t in (q, k, v):
        t.requires_grad_()
    w = torch.randn(4, 3, 32, generator=g)

    def f(q, k, v):
        return (ops.cross_attention(q, k, v, key_mask=mask) * w).double().sum()

    grads = torch.autograd.grad(f(q, k, v), (q, k, v))
    assert all(bool(torch.isfinite(x).all()) for x in grads)
    assert bool((grads[1][mask] == 0).all()) and bool((grads[2][mask] == 0).all()) and bool((grads[0][2:] == 0).all())
    # central differences, h = 2^-6, of sums of 96 fp32 values of order one (roundings of 2^-24 each, a few steps deep): at most
    # 96 * 8 * 2^-24 / 2^-5 = 1.5e-3 from rounding in the worst case; third derivatives below 10 add h^2 / 6 * 10 = 4e-4
    h = 2.0 ** -6
    rng = torch.Generator().manual_seed(2)
    for x, gx, i in ((q, grads[0], 0), (k, grads[1], 1), (v, grads[2], 2)):
        for _ in range(12):
            at = tuple(int(torch.randint(0, s, (1,), generator=rng)) for s in x.shape)
            if i and bool(mask[at[0], at[1]]):
                continue
            args = [t.detach() for t in (q, k, v)]
            d = torch.zeros_like(args[i])
            d[at] = h
            hi = f(*[a + d if n == i else a for n, a in enumerate(args)])
            lo = f(*[a - d if n == i else a for n, a in enumerate(args)])
            assert float(gx[at]) == pytest.approx(float(hi - lo) / (2 * h), abs=2e-3)


@pytest.mark.parametrize("heads,kv_heads,group,tq", [(2, 2, 1, 1), (4, 2, 3, 2)])
def test_shared_prefix_attention_against_single_queries(heads, kv_heads, group, tq):
    g = torch.Generator().manual_seed(3)
    P, S, Smax, D = 2, 4, 6, 8
    B = P * group
    q = torch.randn(B, tq, heads, D, generator=g)
    kp, vp = torch.randn(P, S, kv_heads, D, generator=g), torch.randn(P, S, kv_heads, D, generator=g)
    k, v = torch.randn(B, kv_heads, Smax, D, generator=g).transpose(1, 2), torch.randn(B, kv_heads, Smax, D, generator=g).transpose(1, 2)
    lengths = torch.tensor([tq, 6, 4, 0, 9, 3][:B])
    prefix_lengths = torch.tensor([4, 0])
    out = ops.shared_prefix_attention(q, kp, vp, k, v, lengths, prefix_lengths=prefix_lengths)
    for b in range(B):
        p = b // group
        for t in range(tq):
            own = max(0, min(int(lengths[b]), Smax) - tq + 1 + t)
            for h in range(heads):
                hk = h // (heads // kv_heads)
                keys = [kp[p, j, hk] for j in range(int(prefix_lengths[p]))] + [k[b, j, hk] for j in range(own)]
                values = [vp[p, j, hk] for j in range(int(prefix_lengths[p]))] + [v[b, j, hk] for j in range(own)]
                want = one_query(q[b, t, h], keys, values, 1 / math.sqrt(D))
                assert torch.allclose(out[b, t, h * D:(h + 1) * D].double(), want, rtol=0, atol=64 * 2.0 ** -24)


@pytest.mark.parametrize("kind", [torch.uint8, torch.int8, torch.int16, torch.int32, torch.uint16, torch.uint32])
def test_lengths_of_any_integer_type(kind):
    """Types that do not hold a cache's size, or no negative number: a new token before the first position sees nothing."""
    g = torch.Generator().manual_seed(5)
    q, kp, k = torch.randn(2, 3, 2, 8, generator=g), torch.randn(1, 9, 2, 8, generator=g), torch.randn(2, 300, 2, 8, generator=g)
    lengths, prefix = torch.tensor([1, 7]), torch.tensor([4])
    want = ops.shared_prefix_attention(q, kp, kp, k, k, lengths, prefix_lengths=prefix)
    assert torch.equal(ops.shared_prefix_attention(q, kp, kp, k, k, lengths.to(kind), prefix_lengths=prefix.to(kind)), want)
    assert torch.equal(ops.cross_attention(q, k, k, key_lengths=lengths.to(kind)), ops.cross_attention(q, k, k, key_lengths=lengths))


def test_empty_sizes():
    q, k = torch.randn(2, 3, 2, 8), torch.randn(2, 0, 2, 8)
    assert bool((ops.cross_attention(q, k, k) == 0).all())
    k = torch.randn(2, 4, 2, 8)
    assert ops.cross_attention(q[:, :0], k, k).shape == (2, 0, 16)
    none = k[:, :0]
    own = ops.shared_prefix_attention(q[:, :1], none, none, k, k, torch.tensor([4, 4]))
    assert torch.allclose(own, ops.cross_attention(q[:, :1], k, k), atol=1e-6)
    shared = ops.shared_prefix_attention(q[:, :1], k, k, none, none, torch.tensor([0, 0]))
    assert torch.allclose(shared, own, atol=1e-6)


def test_refusals():
    q, k = torch.randn(4, 3, 4, 8), torch.randn(2, 5, 2, 8)
    bad = [
        (dict(q=q[0], k=k, v=k), "batch, time, heads"),
        (dict(q=q, k=k, v=k[:, :4]), "agree"),
        (dict(q=q[..., :4], k=k, v=k), "head size"),
        (dict(q=q.double(), k=k, v=k), "type"),
        (dict(q=q[:3], k=k, v=k), "multiples"),
        (dict(q=q[:, :, :3], k=k, v=k), "multiples"),
        (dict(q=q, k=k[:0], v=k[:0]), "multiples"),
        (dict(q=q, k=k, v=k, key_lengths=torch.tensor([5])), "key_lengths"),
        (dict(q=q, k=k, v=k, key_lengths=torch.tensor([5.0, 5.0])), "key_lengths"),
        (dict(q=q, k=k, v=k, key_mask=torch.zeros(2, 4, dtype=torch.bool)), "key_mask"),
        (dict(q=q, k=k, v=k, key_mask=torch.zeros(2, 5)), "key_mask"),
    ]
    for kw, match in bad:
        with pytest.raises(ValueError, match=match):
            ops.cross_attention(**kw)
    own, n = torch.randn(4, 6, 2, 8), torch.tensor([1, 2, 3, 4])
    with pytest.raises(ValueError, match="own keys"):
        ops.shared_prefix_attention(q, k, k, own[:3], own[:3], n)
    with pytest.raises(ValueError, match="own keys"):
        ops.shared_prefix_attention(q, k, k, own, own[:, :3], n)
    with pytest.raises(ValueError, match="type"):
        ops.shared_prefix_attention(q, k, k, own.double(), own.double(), n)
    with pytest.raises(ValueError, match="lengths"):
        ops.shared_prefix_attention(q, k, k, own, own, n[:3])
    with pytest.raises(ValueError, match="key_lengths"):
        ops.shared_prefix_attention(q, k, k, own, own, n, prefix_lengths=torch.tensor([1]))
