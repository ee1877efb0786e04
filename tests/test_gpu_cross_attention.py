"""Fused cross attention and shared-prefix attention against a plain statement in 64 bits, with bounds from the roundings made."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

EPS = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}      # half a step, relative
FAST = 2.0 ** -16      # scores up to 2^6 in powers of two, held in fp32 (2^-18 off) and raised by the fast exponential, then summed


def plain(q, k, v, hidden, scale, dout=None):
    """64-bit forward, backward and the error bounds that follow from rounding weights, score gradients and results once each."""
    B, Tq, H, D = q.shape
    M, Tk, Hk, _ = k.shape
    G, rep, e = B // M, H // Hk, EPS[q.dtype]
    qd = q.double().view(M, G, Tq, Hk, rep, D)
    clean = hidden[:, :, None, None]
    kd, vd = k.double().masked_fill(clean, 0.0), v.double().masked_fill(clean, 0.0)
    s = torch.einsum("mgthrd,mshd->mghrts", qd, kd) * scale
    h = hidden[:, None, None, None, None, :]
    s = s.masked_fill(h, -math.inf)
    top = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(top == -math.inf, 0.0, top)).masked_fill(h, 0.0)
    total = p.sum(-1, keepdim=True)
    p = p / torch.where(total == 0, 1.0, total)
    mix = lambda w, x: torch.einsum("mghrts,mshd->mgthrd", w, x).reshape(B, Tq, H, D)   # noqa: E731
    out = mix(p, vd)
    out_err = e * out.abs() + (e + FAST) * mix(p, vd.abs()) + 2.0 ** -25
    if dout is None:
        return out, out_err
    do = dout.double().view(M, G, Tq, Hk, rep, D)
    over = lambda w, x: torch.einsum("mghrts,mgthrd->mshd", w, x)                        # noqa: E731
    dp = torch.einsum("mgthrd,mshd->mghrts", do, vd)
    line = lambda x: torch.einsum("mgthrd,mgthrd->mghrt", do.abs(), x.view(M, G, Tq, Hk, rep, D)).unsqueeze(-1)   # noqa: E731
    delta = torch.einsum("mgthrd,mgthrd->mghrt", do, out.view(M, G, Tq, Hk, rep, D)).unsqueeze(-1)
    ds = p * (dp - delta)
    # delta is computed from the rounded output; fp16 score gradients have an absolute step too, 2^-25 after scaling the largest |do| (or delta / 64) to 8 or more
    ds_err = (e + 2 * FAST) * ds.abs() + p * (line(out_err) + FAST * (dp.abs() + delta.abs())) + (2.0 ** -28 * max(float(dout.abs().max()), float(delta.abs().max()) / 64) if q.dtype == torch.float16 else 0.0)
    ds_err = ds_err.masked_fill(h, 0.0)
    dq, dk, dv = mix(ds, kd) * scale, over(ds, qd) * scale, over(p, do)
    tiny = 2.0 ** -25 if q.dtype == torch.float16 else 1e-30
    dq_err = e * dq.abs() + mix(ds_err, kd.abs()) * scale + FAST * mix(ds.abs(), kd.abs()) * scale + tiny
    dk_err = e * dk.abs() + over(ds_err, qd.abs()) * scale + FAST * over(ds.abs(), qd.abs()) * scale + tiny
    dv_err = e * dv.abs() + (e + 2 * FAST) * over(p, do.abs()) + tiny + (2.0 ** -37 * over((p > 0).double(), do.abs()) if q.dtype == torch.float16 else 0.0)
    return out, out_err, (dq, dk, dv), (dq_err, dk_err, dv_err)


def make(M, G, Tq, Tk, Hk, rep, D, dtype, hide, seed=0, fused=True):
    g = torch.Generator(device="cuda").manual_seed(seed)
    q = (1.5 * torch.randn(M * G, Tq, Hk * rep, D, generator=g, device="cuda")).to(dtype)
    kv = torch.randn(M, Tk, 2, Hk, D, generator=g, device="cuda").to(dtype)
    k, v = (kv[:, :, 0], kv[:, :, 1]) if fused else (kv[:, :, 0].contiguous(), kv[:, :, 1].contiguous())
    lengths = mask = None
    hidden = torch.zeros((M, Tk), dtype=torch.bool, device="cuda")
    if hide in ("lengths", "both"):
        lengths = torch.randint(0, Tk + 1, (M,), generator=g, device="cuda")
        lengths[0] = Tk + 3                                     # beyond the end counts as the end
        if M > 2:
            lengths[2] = 0
        hidden |= torch.arange(Tk, device="cuda")[None] >= lengths[:, None]
    if hide in ("mask", "both"):
        mask = torch.rand((M, Tk), generator=g, device="cuda") < 0.4
        if M > 1:
            mask[1] = True
        hidden |= mask
    k.masked_fill_(hidden[:, :, None, None], float("nan"))
    v.masked_fill_(hidden[:, :, None, None], float("inf"))
    return q, k, v, lengths, mask, hidden


def check(got, want, err, what):
    bad = (got.double() - want).abs() / err
    assert bool(torch.isfinite(got).all()), what
    assert float(bad.max()) <= 1.0, (what, float(bad.max()))


#        M, G, Tq, Tk, Hk, rep, D
SHAPES = [(1, 1, 1, 1, 1, 1, 8), (2, 1, 7, 33, 4, 1, 64), (3, 4, 1, 129, 2, 1, 128), (2, 16, 1, 300, 1, 4, 128), (3, 1, 64, 127, 2, 1, 40),
          (3, 1, 65, 128, 2, 1, 96), (2, 2, 33, 260, 1, 2, 128), (1, 1, 128, 64, 1, 2, 64), (3, 1, 257, 65, 2, 1, 128), (2, 5, 31, 513, 2, 4, 64),
          (1, 1, 300, 1, 3, 1, 72), (1, 3, 130, 1111, 1, 1, 128)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("hide", ["none", "lengths", "mask", "both"])
@pytest.mark.parametrize("shape", SHAPES)
def test_forward(shape, hide, dtype):
    from speech_b200 import ops

    q, k, v, lengths, mask, hidden = make(*shape, dtype, hide)
    out = ops.cross_attention(q, k, v, key_lengths=lengths, key_mask=mask)
    want, err = plain(q, k, v, hidden, 1 / math.sqrt(shape[-1]))
    check(out.view(want.shape), want, err, "out")
    ops.native.check_status()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("hide", ["none", "both"])
@pytest.mark.parametrize("shape", SHAPES)
def test_backward(shape, hide, dtype):
    from speech_b200 import ops

    q, k, v, lengths, mask, hidden = make(*shape, dtype, hide, seed=1)
    dout = torch.randn(q.shape, generator=torch.Generator(device="cuda").manual_seed(5), device="cuda").to(dtype)
    scale = 0.7 / math.sqrt(shape[-1])
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    out = ops.cross_attention(*leaves, key_lengths=lengths, key_mask=mask, scale=scale)
    grads = torch.autograd.grad(out, leaves, dout.flatten(2))
    want, err, dwant, derr = plain(q, k, v, hidden, scale, dout)
    check(out.view(want.shape), want, err, "out")
    for g, w, e, n in zip(grads, dwant, derr, ("dq", "dk", "dv")):
        check(g, w, e, n)
    assert bool((grads[1][hidden] == 0).all()) and bool((grads[2][hidden] == 0).all())
    ops.native.check_status()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("hide", ["none", "lengths", "both", "front"])
@pytest.mark.parametrize("shape", [(1, 1, 100, 2500, 2, 1, 128), (2, 1, 70, 1100, 1, 2, 64), (1, 3, 500, 40, 1, 2, 72), (3, 1, 65, 600, 1, 1, 40),
                                   (38, 1, 65, 2500, 4, 1, 40)])           # 152 tiles: 148 blocks and four clusters
def test_few_tiles_of_long_axes(shape, hide, dtype):
    """Result tiles that several blocks share: parts of the keys that are hidden wholly, lengths that leave blocks without keys."""
    from speech_b200 import ops

    q, k, v, lengths, mask, hidden = make(*shape, dtype, "none" if hide == "front" else hide)
    if hide == "front":
        mask = torch.arange(k.shape[1], device="cuda")[None].expand(k.shape[0], -1) < k.shape[1] - 3
        hidden = mask
        k.masked_fill_(hidden[:, :, None, None], float("nan"))
        v.masked_fill_(hidden[:, :, None, None], float("inf"))
    dout = torch.randn(q.shape, device="cuda", generator=torch.Generator(device="cuda").manual_seed(2)).to(dtype)
    runs = []
    for _ in range(2):
        leaves = [t.detach().requires_grad_() for t in (q, k, v)]
        out = ops.cross_attention(*leaves, key_lengths=lengths, key_mask=mask)
        runs.append((out.detach(),) + torch.autograd.grad(out, leaves, dout.flatten(2)))
    assert all(torch.equal(a, b) for a, b in zip(*runs))
    want, err, dwant, derr = plain(q, k, v, hidden, 1 / math.sqrt(q.shape[3]), dout)
    with torch.no_grad():
        check(ops.cross_attention(q, k, v, key_lengths=lengths, key_mask=mask).view(want.shape), want, err, "out without gradients")
    check(runs[0][0].view(want.shape), want, err, "out")
    for g, w, e, n in zip(runs[0][1:], dwant, derr, ("dq", "dk", "dv")):
        check(g, w, e, n)
    ops.native.check_status()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("tq", [65, 130])                       # one and two row tiles
def test_lengths_that_end_anywhere(tq, dtype):
    """One tile pair per SM of up to 24 key blocks, of which only the last has hidden keys: the warp that clears them runs past all of the others,
    and nothing waits for it until then."""
    from speech_b200 import ops

    M, Tk = 37, 1500
    q, k, v, _, _, hidden = make(M, 1, tq, Tk, 4, 1, 64, dtype, "none", seed=6)
    lengths = torch.tensor([1500 - i if i % 2 else 1 + 40 * i for i in range(M)], device="cuda")
    hidden = torch.arange(Tk, device="cuda")[None] >= lengths[:, None]
    k.masked_fill_(hidden[:, :, None, None], float("nan"))
    v.masked_fill_(hidden[:, :, None, None], float("inf"))
    want, err = plain(q, k, v, hidden, 1 / 8)
    for _ in range(5):
        out = ops.cross_attention(q, k, v, key_lengths=lengths)
        check(out.view(want.shape), want, err, "out")
    ops.native.check_status()


@pytest.mark.parametrize("tq,tk,dim", [(70, 1100, 40), (130, 2050, 72), (259, 700, 104), (2001, 90, 8)])
def test_ragged_tiles_joined_by_clusters(tq, tk, dim):
    """Rows, keys and columns that end inside a tile that several blocks share, where some of a warp's lanes have nothing to join: the same on every
    run, with gradients and without."""
    from speech_b200 import ops

    q, k, v, lengths, mask, hidden = make(1, 1, tq, tk, 1, 1, dim, torch.bfloat16, "none", seed=8)
    dout = torch.randn(q.shape, device="cuda", generator=torch.Generator(device="cuda").manual_seed(9)).to(torch.bfloat16)
    want, err, dwant, derr = plain(q, k, v, hidden, 1 / math.sqrt(dim), dout)
    first = None
    for _ in range(20):
        leaves = [t.detach().requires_grad_() for t in (q, k, v)]
        out = ops.cross_attention(*leaves)
        got = (out.detach(),) + torch.autograd.grad(out, leaves, dout.flatten(2))
        first = first or got
        assert all(torch.equal(a, b) for a, b in zip(got, first))
    check(first[0].view(want.shape), want, err, "out")
    for g, w, e, n in zip(first[1:], dwant, derr, ("dq", "dk", "dv")):
        check(g, w, e, n)
    ops.native.check_status()


@pytest.mark.parametrize("tq", [1, 70, 300])
@pytest.mark.parametrize("tk", [50, 1100])
def test_queries_of_any_value_that_see_nothing(tq, tk):
    """A query that sees no key gets zeros, and no gradient, also where it is infinite or NaN; the other memories' rows are as ever."""
    from speech_b200 import ops

    q, k, v, lengths, mask, hidden = make(3, 2, tq, tk, 2, 1, 64, torch.bfloat16, "both")       # memory 1 is masked wholly, memory 2 has no length
    with torch.no_grad():
        want = ops.cross_attention(q, k, v, key_lengths=lengths, key_mask=mask)
    q = q.clone()
    q[2:, :, 0] = float("inf")
    q[2:, :, 1] = float("nan")
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    out = ops.cross_attention(*leaves, key_lengths=lengths, key_mask=mask)
    with torch.no_grad():
        again = ops.cross_attention(q, k, v, key_lengths=lengths, key_mask=mask)
    grads = torch.autograd.grad(out, leaves, torch.ones_like(out))
    assert torch.equal(out, want) and torch.equal(again, want) and bool((out[2:] == 0).all())
    assert all(bool(torch.isfinite(g).all()) for g in grads) and bool((grads[0][2:] == 0).all())
    assert bool((grads[1][1:] == 0).all()) and bool((grads[2][1:] == 0).all())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("how", ["size", "length", "mask", "both"])
@pytest.mark.parametrize("shape", [(3, 1, 1, 2, 2, 64), (2, 1, 65, 2, 1, 128), (1, 1, 190, 1, 1, 40), (2, 1, 33, 1, 2, 96), (1, 1, 700, 1, 1, 128), (2, 4, 301, 1, 2, 64)])      # M, G, Tq, Hk, rep, D
def test_one_visible_key_has_no_gradient_but_its_value(shape, how, dtype):
    """A softmax over one key is constant: dq and dk are zero, exactly, and the output and dv are the value and the sum of the upstream
    gradients.  Other memories of the same call are as ever."""
    from speech_b200 import ops

    M, G, Tq, Hk, rep, D = shape
    Tk = 1 if how == "size" else 150
    q, k, v, _, _, hidden = make(M, G, Tq, Tk, Hk, rep, D, dtype, "none")
    lengths = mask = None
    rest = slice(M - 1, M) if M > 1 else slice(0, 0)           # the last of several memories keeps all of its keys
    if how in ("length", "both"):
        lengths = torch.full((M,), 1 if how == "length" else 77, device="cuda")
        lengths[rest] = Tk
        hidden = hidden | (torch.arange(Tk, device="cuda")[None] >= lengths[:, None])
    if how in ("mask", "both"):
        mask = torch.arange(Tk, device="cuda")[None].repeat(M, 1) != (149 if how == "mask" else 70)
        mask[rest] = False
        hidden = hidden | mask
    k.masked_fill_(hidden[:, :, None, None], float("nan"))
    v.masked_fill_(hidden[:, :, None, None], float("inf"))
    one = (~hidden).sum(1) == 1
    assert bool(one[0]) and (how == "size" or M == 1 or not bool(one[-1]))
    dout = torch.randn(q.shape, device="cuda", generator=torch.Generator(device="cuda").manual_seed(3)).to(dtype)
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    out = ops.cross_attention(*leaves, key_lengths=lengths, key_mask=mask)
    grads = torch.autograd.grad(out, leaves, dout.flatten(2))
    want, err, dwant, derr = plain(q, k, v, hidden, 1 / math.sqrt(D), dout)
    check(out.view(want.shape), want, err, "out")
    for g, w, e, n in zip(grads, dwant, derr, ("dq", "dk", "dv")):
        check(g, w, e, n)
    assert bool((grads[0].view(M, -1)[one] == 0).all()) and bool((grads[1][one] == 0).all())
    if int(one.sum()) < M:
        assert bool((grads[0].view(M, -1)[~one] != 0).any()) and bool((grads[1][~one] != 0).any())
    ops.native.check_status()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("lead", [3, 4, 5])                    # nats by which a later key leads an early one: less than the maximum may lag
@pytest.mark.parametrize("shape", [(2, 1, 8, 1, 1, 64), (64, 1, 2, 8, 2, 64), (1, 1, 130, 1, 2, 128), (37, 1, 70, 4, 1, 64)])  # M, G, Tq, Hk, rep, D
def test_gradients_of_peaked_rows(shape, lead, dtype):
    """Rows that one key leads: score gradients are differences of nearly equal values, and the output's error, which delta takes on, has to be
    that of a softmax of slightly other weights and not a common factor."""
    from speech_b200 import ops

    M, G, Tq, Hk, rep, D = shape
    q, k, v, _, _, hidden = make(M, G, Tq, 512, Hk, rep, D, dtype, "none", seed=11, fused=False)
    g = torch.Generator(device="cuda").manual_seed(12)
    axis = torch.nn.functional.normalize(torch.randn(D, generator=g, device="cuda"), dim=0) * (8 * D ** 0.5) ** 0.5
    q.copy_(axis + 0.05 * torch.randn(q.shape, generator=g, device="cuda"))
    k.mul_(0.1)
    k[:, 3], k[:, 388] = (axis * 10 / 8).to(dtype), (axis * (10 + lead) / 8).to(dtype)              # scores of 10 and 10 + lead nats, the others' about 0
    dout = torch.randn(q.shape, generator=g, device="cuda").to(dtype)
    e, scale = EPS[dtype], 1 / math.sqrt(D)
    out, _, dwant, _ = plain(q, k, v, hidden, scale, dout)
    qd, kd, vd, do = q.double().view(M, G, Tq, Hk, rep, D), k.double(), v.double(), dout.double().view(M, G, Tq, Hk, rep, D)
    p = torch.softmax(torch.einsum("mgthrd,mshd->mghrts", qd, kd) * scale, -1)
    dp = torch.einsum("mgthrd,mshd->mghrts", do, vd)
    line = torch.einsum("mgthrd,mgthrd->mghrt", do.abs(), out.abs().view(do.shape)).unsqueeze(-1)
    ds = p * (dp - (p * dp).sum(-1, keepdim=True))
    # weights that are rounded by e each and divided by their own sum add up to one, so that delta is off by sum (p' - p) (dp - delta), of
    # |p' - p| <= 2 e p; the output's rounding is made good by its remainder (e^2); fp32 everywhere else
    ds_err = (e + 2 * FAST) * ds.abs() + p * (2 * e * ds.abs().sum(-1, keepdim=True) + (e * e + FAST) * line + FAST * dp.abs())
    ds_err = ds_err + (2.0 ** -28 * float(dout.abs().max()) if dtype == torch.float16 else 0.0)
    dq_err = torch.einsum("mghrts,mshd->mgthrd", ds_err + FAST * ds.abs(), kd.abs()).reshape(q.shape) * scale + e * dwant[0].abs() + 2.0 ** -25
    dk_err = torch.einsum("mghrts,mgthrd->mshd", ds_err + FAST * ds.abs(), qd.abs()) * scale + e * dwant[1].abs() + 2.0 ** -25
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    grads = torch.autograd.grad(ops.cross_attention(*leaves), leaves, dout.flatten(2))
    check(grads[0], dwant[0], dq_err, "dq")
    check(grads[1], dwant[1], dk_err, "dk")
    ops.native.check_status()


@pytest.mark.parametrize("size", [2.0 ** -20, 2.0 ** 12])
def test_fp16_gradients_of_any_size(size):
    """Upstream gradients far from one keep their precision in fp16 (score gradients are scaled)."""
    from speech_b200 import ops

    q, k, v, _, _, hidden = make(1, 1, 130, 700, 2, 1, 64, torch.float16, "none")
    dout = (size * torch.randn(q.shape, device="cuda", generator=torch.Generator(device="cuda").manual_seed(2))).to(torch.float16)
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    out = ops.cross_attention(*leaves)
    grads = torch.autograd.grad(out, leaves, dout.flatten(2))
    _, _, dwant, derr = plain(q, k, v, hidden, 1 / 8, dout)
    for g, w, e, n in zip(grads, dwant, derr, ("dq", "dk", "dv")):
        check(g, w, e, n)


@pytest.mark.parametrize("size", [2.0 ** 8, 2.0 ** 12])
def test_fp16_gradients_of_large_values(size):
    """Values far above one: score gradients (upstream gradient times value) stay within fp16 while they are multiplied."""
    from speech_b200 import ops

    q, k, v, _, _, hidden = make(1, 1, 130, 70, 2, 1, 64, torch.float16, "none")
    v = v * size
    dout = (torch.randn(q.shape, device="cuda", generator=torch.Generator(device="cuda").manual_seed(2)) / size).to(torch.float16)
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    grads = torch.autograd.grad(ops.cross_attention(*leaves), leaves, dout.flatten(2))
    _, _, dwant, derr = plain(q, k, v, hidden, 1 / 8, dout)
    for g, w, e, n in zip(grads, dwant, derr, ("dq", "dk", "dv")):
        check(g, w, e, n)


@pytest.mark.parametrize("tq,tk", [(5, 2), (70, 200), (130, 700)])
@pytest.mark.parametrize("size", [200.0, 4000.0, 60000.0])
def test_fp16_gradients_of_values_that_cancel(size, tq, tk):
    """Values of both signs whose weighted mean is small: delta cancels and dp does not, and score gradients still stay within fp16 (their bound is
    that of |do| |v|, whatever the sum)."""
    from speech_b200 import ops

    g = torch.Generator(device="cuda").manual_seed(0)
    q = (0.01 * torch.randn(1, tq, 2, 128, generator=g, device="cuda")).half()
    k = (0.01 * torch.randn(1, tk, 2, 128, generator=g, device="cuda")).half()
    sign = 1.0 - 2.0 * (torch.arange(tk, device="cuda") % 2)
    v = (size * sign).view(1, tk, 1, 1).expand(1, tk, 2, 128).half()
    mask = torch.zeros((1, tk + 1), dtype=torch.bool, device="cuda")
    mask[:, tk] = True                                        # a hidden infinity has no part in the bound
    k, v = torch.cat([k, k[:, :1]], 1), torch.cat([v, torch.full_like(v[:, :1], float("inf"))], 1)
    dout = (torch.ones(q.shape, device="cuda") / max(1.0, size / 200)).half()
    hidden = mask
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    grads = torch.autograd.grad(ops.cross_attention(*leaves, key_mask=mask), leaves, dout.flatten(2))
    _, _, dwant, derr = plain(q, k, v, hidden, 1 / 128 ** 0.5, dout)
    # besides plain()'s bounds: ds has an absolute step where the values' size sets its scale: the factor is at least 2^3 / (|do| sqrt(D) |v| / 2^12)
    # for a power of two, the step 2^-25 over that
    step = 2.0 ** -25 * float(dout.abs().max()) * 128 ** 0.5 * size * 128 ** 0.5 / 2.0 ** 12 / 2.0 ** 3
    dq_more = step * k.double().abs().sum(1, keepdim=True) / 128 ** 0.5
    dk_more = step * q.double().abs().sum(1, keepdim=True) / 128 ** 0.5
    check(grads[0], dwant[0], derr[0] + dq_more, "dq")
    check(grads[1], dwant[1], derr[1] + dk_more, "dk")
    check(grads[2], dwant[2], derr[2], "dv")
    ops.native.check_status()


def test_gradients_against_differences():
    from speech_b200 import ops

    q, k, v, lengths, mask, hidden = make(2, 2, 40, 90, 1, 2, 64, torch.bfloat16, "none")
    w = torch.randn(q.shape, device="cuda", generator=torch.Generator(device="cuda").manual_seed(4)).to(torch.bfloat16)
    leaves = [t.detach().contiguous().requires_grad_() for t in (q, k, v)]
    grads = torch.autograd.grad(ops.cross_attention(*leaves), leaves, w.flatten(2))
    for i in range(3):
        d = torch.randn(leaves[i].shape, device="cuda", generator=torch.Generator(device="cuda").manual_seed(i)).double()
        h = 2.0 ** -10

        def f(sign):
            args = [x.detach().double() for x in leaves]
            args[i] = args[i] + sign * h * d
            s = torch.einsum("mgthrd,mshd->mghrts", args[0].view(2, 2, 40, 1, 2, 64), args[1]) / 8
            return (torch.einsum("mghrts,mshd->mgthrd", torch.softmax(s, -1), args[2]).reshape(w.shape) * w.double()).sum()

        slope, got = float((f(1) - f(-1)) / (2 * h)), float((grads[i].double() * d).sum())
        # every gradient element is off by a few bf16 half steps of its own size and of the terms it sums (factor 8), at random signs against d
        assert abs(got - slope) <= 8 * 2.0 ** -8 * float((grads[i].double() * d).norm()) + 1e-4 * abs(slope)


def test_strides_and_unaligned_inputs():
    """Heads-first caches, slices at odd offsets, broadcast memories: the same results as contiguous copies."""
    from speech_b200 import ops

    for Tq in (3, 140):
        q, k, v, _, mask, _ = make(2, 2, Tq, 200, 2, 2, 64, torch.bfloat16, "mask", fused=False)
        want = ops.cross_attention(q, k, v, key_mask=mask)
        qh, kh, vh = (t.transpose(1, 2).contiguous().transpose(1, 2) for t in (q, k, v))
        assert torch.equal(ops.cross_attention(qh, kh, vh, key_mask=mask), want)
        wide = torch.zeros(k.shape[:3] + (67,), dtype=k.dtype, device="cuda")
        wide[..., 3:] = k
        odd = wide[..., 3:]
        assert odd.data_ptr() % 16 and torch.equal(ops.cross_attention(q, odd, v, key_mask=mask), want)
        wide_mask = torch.zeros((2, 401), dtype=torch.bool, device="cuda")
        wide_mask[:, 1::2] = mask
        assert torch.equal(ops.cross_attention(q, k, v, key_mask=wide_mask[:, 1::2]), want)
        one = k[:1].nan_to_num().expand(2, -1, -1, -1)
        assert torch.equal(ops.cross_attention(q, one, one), ops.cross_attention(q, one.contiguous(), one.contiguous()))
        longs = torch.tensor([150, 2 ** 40], device="cuda")
        assert torch.equal(ops.cross_attention(q, k, v, key_lengths=longs, key_mask=mask),
                           ops.cross_attention(q, k, v, key_lengths=torch.tensor([150, 200], dtype=torch.int32, device="cuda"), key_mask=mask))


@pytest.mark.parametrize("tq", [1, 3, 140])
def test_dense_views_that_the_kernels_cannot_address(tq):
    """Views that count as contiguous and still start off a 16-byte boundary, or have odd strides of axes of size one."""
    from speech_b200 import ops

    def at_one(t):                                             # the same values, dense, one element into their storage
        flat = torch.zeros(t.numel() + 1, dtype=t.dtype, device="cuda")
        flat[1:] = t.flatten()
        return flat[1:].view(t.shape)

    def odd(t):                                                # [1, 1, H, D] out of a projection of odd width
        wide = torch.zeros((1, 1, t.shape[2] * t.shape[3] + 3), dtype=t.dtype, device="cuda")
        wide[..., :-3] = t.flatten(2)
        return wide.as_strided(t.shape, (wide.shape[2], wide.shape[2], t.shape[3], 1))

    for M, tk, move in ((2, 200, at_one), (1, 1, odd)) if tq == 1 else ((2, 200, at_one),):
        q, k, v, _, _, _ = make(M, 1, tq, tk, 2, 1, 64, torch.bfloat16, "none", fused=False)
        moved = [move(t) for t in (q, k, v)]
        assert all(t.is_contiguous() and torch.equal(t, u) for t, u in zip(moved, (q, k, v)))
        results = []
        for tensors in [(q, k, v)] + [tuple(m if i == j else t for j, (t, m) in enumerate(zip((q, k, v), moved))) for i in range(3)] + [moved]:
            leaves = [t.detach().requires_grad_() for t in tensors]
            out = ops.cross_attention(*leaves)
            with torch.no_grad():
                both = [ops.shared_prefix_attention(*tensors, *tensors[1:], torch.full((M,), tk, device="cuda"))] if tq <= 3 else []
            results.append([out.detach(), ops.cross_attention(*tensors), *both, *torch.autograd.grad(out, leaves, torch.ones_like(out))])
        for r in results[1:]:
            assert all(torch.equal(a, b) for a, b in zip(r, results[0]))
    ops.native.check_status()


@pytest.mark.parametrize("kind", [torch.uint8, torch.int8, torch.int16, torch.int32, torch.uint16, torch.uint32])
def test_lengths_of_any_integer_type(kind):
    from speech_b200 import ops

    for tq in (3, 70):
        q, k, v, _, _, _ = make(2, 1, tq, 300, 2, 1, 64, torch.bfloat16, "none")
        lengths = torch.tensor([1, 100], device="cuda")
        assert torch.equal(ops.cross_attention(q, k, v, key_lengths=lengths.to(kind)), ops.cross_attention(q, k, v, key_lengths=lengths))
        want = ops.shared_prefix_attention(q, k, v, k, v, lengths, prefix_lengths=lengths)
        assert torch.equal(ops.shared_prefix_attention(q, k, v, k, v, lengths.to(kind), prefix_lengths=lengths.to(kind)), want)
        if kind in (torch.int8, torch.int16, torch.int32):
            none = torch.tensor([-1, -100], device="cuda")
            assert bool((ops.cross_attention(q, k, v, key_lengths=none.to(kind)) == 0).all())


def test_partial_gradients_and_determinism():
    from speech_b200 import ops

    q, k, v, lengths, mask, _ = make(2, 3, 50, 333, 2, 2, 64, torch.bfloat16, "both")
    dout = torch.randn(q.shape, device="cuda").to(torch.bfloat16).flatten(2)

    def grads(want):
        leaves = [t.detach().requires_grad_(w) for t, w in zip((q, k, v), want)]
        out = ops.cross_attention(*leaves, key_lengths=lengths, key_mask=mask)
        return torch.autograd.grad(out, [x for x in leaves if x.requires_grad], dout)

    full, again = grads((True, True, True)), grads((True, True, True))
    assert all(torch.equal(a, b) for a, b in zip(full, again))
    assert torch.equal(grads((True, False, False))[0], full[0])
    assert torch.equal(grads((False, True, False))[0], full[1])
    assert torch.equal(grads((False, False, True))[0], full[2])
    # a gradient that arrives transposed, and one that is a broadcast scalar
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    out = ops.cross_attention(*leaves, key_lengths=lengths, key_mask=mask)
    odd = dout.transpose(0, 1).contiguous().transpose(0, 1)
    assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(out, leaves, odd, retain_graph=True), full))
    out.sum().backward()
    assert bool(torch.isfinite(leaves[0].grad).all())


def test_double_backward_is_refused():
    from speech_b200 import ops

    q = torch.randn(1, 3, 2, 64, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    (g,) = torch.autograd.grad(ops.cross_attention(q, q, q).float().sum(), q, create_graph=True)
    with pytest.raises(RuntimeError):
        g.float().sum().backward()


def test_forward_mode_derivatives_are_there_or_refused():
    """A dual tensor has no requires_grad; its tangent must not be lost."""
    import torch.autograd.forward_ad as forward_ad

    from speech_b200 import ops

    q, k, v, lengths, _, hidden = make(2, 1, 5, 40, 2, 1, 64, torch.bfloat16, "lengths")
    g = torch.Generator(device="cuda").manual_seed(3)
    tangents = [torch.randn(t.shape, generator=g, device="cuda").to(torch.bfloat16) for t in (q, k, v)]
    # 64-bit: derivative along the tangents from three gradients
    dout = torch.randn(q.shape, generator=g, device="cuda").to(torch.bfloat16)
    _, _, (dq, dk, dv), _ = plain(q, k, v, hidden, 1 / 8, dout)
    want = sum(float((d * t.double()).sum()) for d, t in zip((dq, dk, dv), tangents))
    size = sum(float((d * t.double()).norm()) for d, t in zip((dq, dk, dv), tangents))
    with forward_ad.dual_level():
        duals = [forward_ad.make_dual(t, d) for t, d in zip((q, k, v), tangents)]
        out = forward_ad.unpack_dual(ops.cross_attention(*duals, key_lengths=lengths))
        assert out.tangent is not None
        # the result's tangent is rounded to bf16: by at most 2^-8 of itself at random signs, as many as there are elements (factor 6)
        got = float((out.tangent.double() * dout.flatten(2).double()).sum())
        assert abs(got - want) <= 6 * 2.0 ** -8 * (float((out.tangent.double() * dout.flatten(2).double()).norm()) + size)
        for i in range(3):
            args = [duals[j] if i == j else t for j, t in enumerate((q, k, v))]
            assert forward_ad.unpack_dual(ops.cross_attention(*args, key_lengths=lengths)).tangent is not None
            with pytest.raises(RuntimeError, match="forward-mode"):
                ops.shared_prefix_attention(*args, k, v, torch.tensor([3, 9], device="cuda"))
        assert forward_ad.unpack_dual(ops.cross_attention(q, k, v, key_lengths=lengths)).tangent is None
    _, tangent = torch.func.jvp(lambda x: ops.cross_attention(x, k, v, key_lengths=lengths), (q,), (tangents[0],))
    assert float(tangent.float().abs().max()) > 0


def test_what_backward_needs_is_seen_by_autograd():
    """Everything kept for the backward pass goes through saved variables: hooks move it, and it is freed with the graph though the output lives."""
    from speech_b200 import ops

    q, k, v, lengths, _, _ = make(4, 2, 500, 300, 4, 1, 64, torch.bfloat16, "lengths")
    dout = torch.randn(q.shape, device="cuda").to(torch.bfloat16).flatten(2)
    size = q.numel() * q.element_size()

    def run():
        leaves = [t.detach().requires_grad_() for t in (q, k, v)]
        before = torch.cuda.memory_allocated()
        out = ops.cross_attention(*leaves, key_lengths=lengths)
        after = torch.cuda.memory_allocated() - before
        grads = torch.autograd.grad(out, leaves, dout)
        return out, grads, after, torch.cuda.memory_allocated() - before - sum(g.numel() * g.element_size() for g in grads)

    out, grads, _, left = run()
    assert left < 1.25 * size                               # the output alone
    with torch.autograd.graph.save_on_cpu():
        again, moved, held, _ = run()
    assert held < 1.25 * size
    assert torch.equal(again, out) and all(torch.equal(a, b) for a, b in zip(moved, grads))

    from torch.utils.checkpoint import checkpoint

    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    once = checkpoint(lambda *t: ops.cross_attention(*t, key_lengths=lengths), *leaves, use_reentrant=False)
    assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(once, leaves, dout), grads))


def test_other_stream_and_captured_graphs():
    """Two captured graphs and an eager call in between, on inputs that change between replays."""
    from speech_b200 import ops

    cases = [make(2, 2, 1, 700, 2, 2, 128, torch.bfloat16, "lengths"), make(2, 1, 200, 300, 2, 2, 64, torch.bfloat16, "lengths")]
    side = torch.cuda.Stream()
    graphs, outs = [], []

    def call(c):
        leaves = [t.detach().requires_grad_() for t in c[:3]]
        out = ops.cross_attention(*leaves, key_lengths=c[3])
        return (out.detach(),) + torch.autograd.grad(out, leaves, torch.ones_like(out))

    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for c in cases:
            first = call(c)
    torch.cuda.current_stream().wait_stream(side)
    for c in cases:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(call(c))
        graphs.append(graph)
    for c, seed in zip(cases, (7, 8)):
        for t in c[:3]:
            t.copy_(torch.randn(t.shape, device="cuda", generator=torch.Generator(device="cuda").manual_seed(seed)))
        c[3].copy_(torch.tensor([100, 250], device="cuda"))
    graphs[0].replay()
    graphs[1].replay()
    want = [[x.clone() for x in call(c)] for c in cases]
    graphs[0].replay()
    torch.cuda.synchronize()
    for a, b in zip(outs, want):
        assert all(torch.equal(x, y) for x, y in zip(a, b))
    ops.native.check_status()


# ------------------------------------------------------------------------------------------------ shared prefix
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("shape", [(1, 1, 1, 1, 8, 1, 1, 8), (1, 4, 1, 129, 17, 8, 2, 128), (3, 16, 1, 700, 65, 2, 2, 128), (2, 3, 5, 40, 300, 2, 4, 64),
                                   (2, 40, 2, 333, 16, 1, 1, 40), (5, 1, 1, 2000, 1000, 1, 4, 96)])
def test_shared_prefix(shape, dtype):
    from speech_b200 import ops

    P, G, Tq, S, Smax, Hk, rep, D = shape
    B = P * G
    g = torch.Generator(device="cuda").manual_seed(0)
    r = lambda *s: torch.randn(s, generator=g, device="cuda").to(dtype)      # noqa: E731
    q, kp, vp, k, v = 1.5 * r(B, Tq, Hk * rep, D), r(P, S, Hk, D), r(P, S, Hk, D), r(B, Hk, Smax, D).transpose(1, 2), r(B, Hk, Smax, D).transpose(1, 2)
    plen = torch.randint(0, S + 1, (P,), generator=g, device="cuda")
    plen[0] = S
    lens = torch.randint(0, Smax + 1, (B,), generator=g, device="cuda")
    lens[B // 2] = Smax + 5
    lens[0] = Tq - 1                                            # the first new token sees the prompt alone
    for b in range(B):                                          # what lies behind the lengths is garbage
        k[b, int(lens[b]):] = float("nan")
        v[b, int(lens[b]):] = float("inf")
    for p in range(P):
        kp[p, int(plen[p]):] = float("inf")
        vp[p, int(plen[p]):] = float("nan")
    out = ops.shared_prefix_attention(q, kp, vp, k, v, lens, prefix_lengths=plen).view(B, Tq, Hk * rep, D)
    for b in range(B):
        n, own = int(plen[b // G]), min(int(lens[b]), Smax)
        for t in range(Tq):
            upto = max(0, own - Tq + 1 + t)
            kk = torch.cat([kp[b // G, :n], k[b, :upto]])[None]
            vv = torch.cat([vp[b // G, :n], v[b, :upto]])[None]
            if kk.shape[1] == 0:
                assert bool((out[b, t] == 0).all())
                continue
            want, err = plain(q[b:b + 1, t:t + 1], kk, vv, torch.zeros((1, kk.shape[1]), dtype=torch.bool, device="cuda"), 1 / math.sqrt(D))
            check(out[b:b + 1, t:t + 1], want, err, (b, t))


def test_shared_prefix_refuses_gradients_and_takes_empty_caches():
    from speech_b200 import ops

    q, k = torch.randn(4, 1, 2, 64, device="cuda", dtype=torch.bfloat16), torch.randn(2, 9, 2, 64, device="cuda", dtype=torch.bfloat16)
    own, n = torch.randn(4, 5, 2, 64, device="cuda", dtype=torch.bfloat16), torch.tensor([1, 2, 3, 5], device="cuda")
    with pytest.raises(RuntimeError, match="no backward"):
        ops.shared_prefix_attention(q.requires_grad_(), k, k, own, own, n)
    with torch.no_grad():
        ops.shared_prefix_attention(q, k, k, own, own, n)
    q = q.detach()
    a = ops.shared_prefix_attention(q, k[:, :0], k[:, :0], own, own, n)
    b = ops.cross_attention(q, own, own, key_lengths=n)
    # one is the plain form in fp32, the other the kernel: both within a bf16 step of the same value
    assert bool(((a.float() - b.float()).abs() <= 2.0 ** -6 * (1 + b.float().abs())).all())


def test_run_of_the_operators_together():
    """A group of answers per memory: decoding steps over the shared states and the shared prompt, teacher forcing over the same states,
    policy loss and gradients down to queries, keys and values."""
    from speech_b200 import ops

    M, G, T, Tk, H, D, V = 2, 4, 6, 90, 4, 64, 130
    q, k, v, lengths, _, hidden = make(M, G, T, Tk, H, 1, D, torch.bfloat16, "lengths", fused=False)
    full = ops.cross_attention(q, k, v, key_lengths=lengths)
    steps = torch.cat([ops.cross_attention(q[:, t:t + 1], k, v, key_lengths=lengths) for t in range(T)], dim=1)
    want, err = plain(q, k, v, hidden, 1 / 8)
    check(full.view(want.shape), want, err, "all at once")
    check(steps.view(want.shape), want, err, "one at a time")
    own = torch.randn(M * G, T, H, D, device="cuda").to(torch.bfloat16)
    both = ops.shared_prefix_attention(q[:, -1:], k, v, own, own, torch.full((M * G,), T, device="cuda"), prefix_lengths=lengths)
    assert bool(torch.isfinite(both).all())
    head = (0.1 * torch.randn(V, H * D, device="cuda", generator=torch.Generator(device="cuda").manual_seed(1))).to(torch.bfloat16)
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    logits = torch.nn.functional.linear(ops.cross_attention(*leaves, key_lengths=lengths), head)
    targets = torch.randint(0, V, (M * G, T), device="cuda")
    mask = torch.ones((M * G, T), dtype=torch.bool, device="cuda")
    with torch.no_grad():
        old = torch.log_softmax(logits.double(), -1).gather(-1, targets.unsqueeze(-1)).squeeze(-1).float()
    loss, logp = ops.policy_loss(logits, targets, mask, old, torch.randn(M * G, device="cuda"), ref_logp=old, kl_beta=0.04)
    loss.backward()
    assert torch.allclose(logp, old, atol=1e-5) and all(bool(torch.isfinite(x.grad).all()) and float(x.grad.abs().max()) > 0 for x in leaves)
    pref, _ = ops.preference_loss(logits.detach().requires_grad_(), targets, mask, old)
    assert abs(float(pref) - math.log(2)) < 1e-4
    ops.native.check_status()


def test_offsets_beyond_32_bits():
    """Memories and caches whose rows lie more than 2^31 elements apart."""
    from speech_b200 import ops

    q, k, v, lengths, mask, _ = make(2, 2, 70, 150, 2, 1, 64, torch.bfloat16, "both", fused=False)
    far = torch.empty(2 ** 31 + 2 ** 20, dtype=torch.bfloat16, device="cuda")
    apart = lambda t, at: far.as_strided(t.shape, (2 ** 31 + 2 ** 17,) + t.stride()[1:], at).copy_(t)       # noqa: E731

    def run(k, v, mask):
        leaves = [t.detach().requires_grad_() for t in (q, k, v)]
        out = ops.cross_attention(*leaves, key_lengths=lengths, key_mask=mask)
        with torch.no_grad():
            step = ops.cross_attention(q[:, :1], k, v, key_lengths=lengths, key_mask=mask)
            both = ops.shared_prefix_attention(q[:2, :1], k, v, k, v, lengths.clamp(max=140), prefix_lengths=lengths)
        return [t.detach().contiguous().view(torch.int16) for t in (out, step, both) + torch.autograd.grad(out, leaves, torch.ones_like(out))]

    clean = lambda t: t.nan_to_num(1.0, 1.0, 1.0)           # noqa: E731
    names = ("out", "step", "both", "dq", "dk", "dv")
    for what, x, y, m in (("hidden garbage", k, v, mask), ("all but the lengths seen", clean(k), clean(v), None)):
        near, at = run(x, y, m), run(apart(x, 0), apart(y, 2 ** 16), m)
        assert [n for n, a, b in zip(names, near, at) if not torch.equal(a, b)] == [], what
    ops.native.check_status()


def test_calls_from_two_threads():
    import threading

    from speech_b200 import ops

    cases, results = [make(2, 2, 130, t, 2, 1, 64, torch.float16, "lengths", seed=t) for t in (300, 77)], [[], []]

    def call(c):
        leaves = [t.detach().requires_grad_() for t in c[:3]]
        out = ops.cross_attention(*leaves, key_lengths=c[3])
        with torch.no_grad():
            step = ops.cross_attention(c[0][:, :1], c[1], c[2], key_lengths=c[3])
        return (out, step) + torch.autograd.grad(out, leaves, torch.ones_like(out))

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
    ops.native.check_status()
