"""Measured cases of the post-training operators: attention of a decoder over an encoder's states (training, and one token per
call with beams or sampled groups that share the states), attention of a sampled group over a prompt that all of it shares, and
the policy and preference losses that turn the logits of such a batch into a scalar and the logits' gradient.

``run`` computes a case with elementary torch operations, or, where ``own`` is set, through ``speech_b200.ops``.
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


# ------------------------------------------------------------------------------------------------ cases
def _cross(name, train, memories, group, tq, tk, heads, kv_heads, dim, dtype, hidden):
    return {"name": name, "op": "cross", "train": train, "memories": memories, "group": group, "tq": tq, "tk": tk, "heads": heads,
            "kv_heads": kv_heads, "dim": dim, "dtype": dtype, "hidden": hidden}


def _prefix(name, prompts, group, tq, prefix, own_max, heads, kv_heads, dim, dtype):
    return {"name": name, "op": "prefix", "prompts": prompts, "group": group, "tq": tq, "prefix": prefix, "own_max": own_max,
            "heads": heads, "kv_heads": kv_heads, "dim": dim, "dtype": dtype}


def _policy(name, seqs, steps, books, vocab, dtype, kl):
    return {"name": name, "op": "policy", "seqs": seqs, "steps": steps, "books": books, "vocab": vocab, "dtype": dtype, "kl": kl}


def _preference(name, pairs, steps, books, vocab, dtype, loss):
    return {"name": name, "op": "preference", "pairs": pairs, "steps": steps, "books": books, "vocab": vocab, "dtype": dtype, "loss": loss}


def listed():
    return [
        # the smallest training step of a decoder over encoder states: a unit-test batch, where only latency counts
        _cross("cross_train_tiny", True, 2, 1, 7, 33, 4, 4, 64, "bf16", "lengths"),
        # a training batch of the attention encoder-decoder (8 heads of 128): transcripts against up to 40 s of 80 ms frames
        _cross("cross_train_utterances", True, 32, 1, 187, 501, 8, 8, 128, "bf16", "lengths"),
        # long-form training: full-length transcripts against ten minutes of frames
        _cross("cross_train_long", True, 4, 1, 1024, 7500, 8, 8, 128, "bf16", "none"),
        # sampled groups scored against shared states, shared key heads, frames hidden one by one and one memory hidden wholly
        _cross("cross_train_groups", True, 3, 4, 301, 1111, 16, 4, 64, "fp16", "mask"),
        # one token of one utterance: the latency of greedy decoding (30 s of frames)
        _cross("cross_step_one", False, 1, 1, 1, 375, 8, 8, 128, "bf16", "none"),
        # one token of every beam of a batch: four beams share the states of their utterance
        _cross("cross_step_beams", False, 16, 4, 1, 501, 8, 8, 128, "bf16", "lengths"),
        # one token for four samples of one short prompt
        _prefix("prefix_step_small", 1, 4, 1, 129, 17, 16, 8, 128, "bf16"),
        # one token for sixteen samples of each of eight prompts with a long audio context
        _prefix("prefix_step_groups", 8, 16, 1, 1500, 511, 16, 8, 128, "bf16"),
        # a unit-test batch of the policy loss
        _policy("policy_tiny", 3, 9, 8, 2024, "bf16", True),
        # four prompts with eight samples each, 20 s of codec frames in eight codebooks
        _policy("policy_codes", 32, 430, 8, 2024, "bf16", True),
        # eight pairs of chosen and rejected generations of 10 s
        _preference("preference_codes", 8, 215, 8, 2024, "bf16", "dpo"),
        # four pairs of text answers over a language model's vocabulary
        _preference("preference_text", 4, 127, 1, 151936, "bf16", "ipo"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    most = {"cross_train": 4 * 1024 * 7500 * 8 * 128, "cross_step": 16 * 501 * 8 * 128 * 2, "prefix": 8 * 1500 * 8 * 128 * 2 + 128 * 511 * 8 * 128,
            "rows": 32 * 430 * 8 * 2024}
    kind = rng.choice(["cross_train", "cross_train", "cross_step", "prefix", "policy", "preference"])
    while True:
        dtype = rng.choice(["bf16", "bf16", "fp16"])
        kv_heads, rep, dim = rng.choice([1, 2, 4, 8, 12]), rng.choice([1, 1, 2, 4]), rng.choice([64, 64, 128, 128, 40, 96])
        if kind == "cross_train":
            memories, group, tq, tk = _log_int(rng, 1, 32), rng.choice([1, 1, 2, 5]), _log_int(rng, 1, 1500), _log_int(rng, 1, 7500)
            if memories * group * tq * tk * kv_heads * rep * dim <= most[kind]:
                return _cross("", True, memories, group, tq, tk, kv_heads * rep, kv_heads, dim, dtype, rng.choice(["none", "lengths", "mask"]))
        elif kind == "cross_step":
            memories, group, tq, tk = _log_int(rng, 1, 64), rng.choice([1, 2, 4, 7, 16]), rng.choice([1, 1, 1, 3]), _log_int(rng, 1, 7500)
            if memories * tk * kv_heads * dim <= most[kind]:
                return _cross("", False, memories, group, tq, tk, kv_heads * rep, kv_heads, dim, dtype, rng.choice(["none", "lengths", "mask"]))
        elif kind == "prefix":
            prompts, group, tq = _log_int(rng, 1, 16), _log_int(rng, 1, 32), rng.choice([1, 1, 1, 2, 5])
            prefix, own_max = _log_int(rng, 1, 6000), _log_int(rng, 8, 1100)
            if (prompts * prefix + prompts * group * own_max) * kv_heads * dim <= most[kind]:
                return _prefix("", prompts, group, tq, prefix, own_max, kv_heads * rep, kv_heads, dim, dtype)
        else:
            seqs, steps, books = 2 * _log_int(rng, 1, 24), _log_int(rng, 1, 700), rng.choice([1, 4, 8])
            vocab, dtype = _log_int(rng, 130, 152000), rng.choice(["bf16", "bf16", "fp16", "fp32"])
            if seqs * steps * books * vocab <= most["rows"] // (2 if dtype == "fp32" else 1):
                if kind == "policy":
                    return _policy("", seqs, steps, books, vocab, dtype, rng.choice([True, False]))
                return _preference("", seqs // 2, steps, books, vocab, dtype, rng.choice(["dpo", "ipo", "rpo_sq"]))


def _spread(n, lo, hi):
    """``n`` lengths in [lo, hi] in no order, the longest among them: the ragged batch of a case (the same for every seed)."""
    return [hi if i == n // 2 else lo + (i * 7919 + 13) * 104729 % (hi - lo + 1) for i in range(n)]


def _key_lengths(c):
    return _spread(c["memories"], max(1, c["tk"] * 2 // 5), c["tk"]) if c["hidden"] == "lengths" else [c["tk"]] * c["memories"]


def _prefix_lengths(c):
    return _spread(c["prompts"], max(1, c["prefix"] * 3 // 5), c["prefix"])


def _own_lengths(c):
    return _spread(c["prompts"] * c["group"], min(c["tq"], c["own_max"]), c["own_max"])


def _steps(c):
    n = 2 * c["pairs"] if c["op"] == "preference" else c["seqs"]
    return n, _spread(n, max(1, c["steps"] // 2), c["steps"])


# ------------------------------------------------------------------------------------------------ inputs
def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    dt = DTYPES[case["dtype"]]

    def normal(*shape, scale=1.0):
        return (torch.randn(shape, generator=g, device=dev) * scale).to(dt)

    s = {"case": dict(case)}
    if case["op"] == "cross":
        B, H, D = case["memories"] * case["group"], case["heads"], case["dim"]
        s["q"] = normal(B, case["tq"], H, D, scale=1.5)
        kv = normal(case["memories"], case["tk"], 2, case["kv_heads"], D)      # keys and values come out of one projection
        s["k"], s["v"] = kv[:, :, 0], kv[:, :, 1]
        s["lengths"] = s["hidden"] = None
        if case["hidden"] == "lengths":
            s["lengths"] = torch.tensor(_key_lengths(case), dtype=torch.int32, device=dev)
        elif case["hidden"] == "mask":
            s["hidden"] = torch.rand((case["memories"], case["tk"]), generator=g, device=dev) < 0.3
            if case["memories"] > 2:
                s["hidden"][1] = True
        if case["train"]:
            s["dout"] = normal(B, case["tq"], H * D)
    elif case["op"] == "prefix":
        P, B, H, Hk, D = case["prompts"], case["prompts"] * case["group"], case["heads"], case["kv_heads"], case["dim"]
        s["q"] = normal(B, case["tq"], H, D, scale=1.5)
        # the caches of a language model hold [row, head, position, dim]
        s["kp"], s["vp"] = normal(P, Hk, case["prefix"], D).transpose(1, 2), normal(P, Hk, case["prefix"], D).transpose(1, 2)
        s["k"], s["v"] = normal(B, Hk, case["own_max"], D).transpose(1, 2), normal(B, Hk, case["own_max"], D).transpose(1, 2)
        s["prefix_lengths"] = torch.tensor(_prefix_lengths(case), dtype=torch.int32, device=dev)
        s["lengths"] = torch.tensor(_own_lengths(case), dtype=torch.int32, device=dev)
    else:
        n, steps = _steps(case)
        T, C, V = case["steps"], case["books"], case["vocab"]
        # gradients in fp16 are computed of the loss times a scale that keeps them in the type's range
        s["grad"] = torch.tensor(1024.0 if case["dtype"] == "fp16" else 1.0, device=dev)
        s["logits"] = normal(n, T, C, V, scale=2.0)
        s["targets"] = torch.randint(0, V, (n, T, C), generator=g, device=dev)
        s["mask"] = torch.arange(T, device=dev)[None, :] < torch.tensor(steps, device=dev)[:, None]
        m = s["logits"].amax(-1).float()
        total = torch.stack([torch.exp(s["logits"][i].float() - m[i].unsqueeze(-1)).sum(-1) for i in range(n)])
        logp = s["logits"].gather(-1, s["targets"].unsqueeze(-1)).squeeze(-1).float() - m - total.log()
        # the policy that sampled the batch and the frozen one are near the one that is trained
        s["ref"] = logp + 0.1 * torch.randn(logp.shape, generator=g, device=dev)
        if case["op"] == "policy":
            s["old"] = logp + 0.15 * torch.randn(logp.shape, generator=g, device=dev)
            s["advantages"] = torch.randn(n, generator=g, device=dev)
            if not case["kl"]:
                s["ref"] = None
        else:
            s["gap"] = torch.rand(n // 2, generator=g, device=dev) if case["loss"] == "rpo_sq" else None
    return s


# ------------------------------------------------------------------------------------------------ plain forms
CLIP, KL_BETA, BETA = 0.2, 0.04, 0.1


def _softmax(scores):
    """Softmax over the last axis; a row in which everything is hidden has no weights."""
    m = scores.amax(-1, keepdim=True)
    e = torch.exp(scores - torch.where(m == -math.inf, torch.zeros_like(m), m))
    total = e.sum(-1, keepdim=True)
    return e / torch.where(total == 0, torch.ones_like(total), total)


def _plain_cross(s):
    c = s["case"]
    M, G, Tq, Tk, Hk, D = c["memories"], c["group"], c["tq"], c["tk"], c["kv_heads"], c["dim"]
    rep, dt, scale = c["heads"] // Hk, s["q"].dtype, 1.0 / math.sqrt(D)

    def rows(x):        # [B, Tq, H, D] -> [M, Hk, G * rep * Tq, D]: the rows that read the same keys, together
        return x.float().view(M, G, Tq, Hk, rep, D).permute(0, 3, 1, 4, 2, 5).reshape(M, Hk, G * rep * Tq, D)

    def back(x):
        return x.view(M, Hk, G, rep, Tq, D).permute(0, 2, 4, 1, 3, 5).reshape(M * G, Tq, Hk * rep, D).to(dt)

    q, k, v = rows(s["q"]), s["k"].float().transpose(1, 2), s["v"].float().transpose(1, 2)
    scores = torch.matmul(q, k.transpose(-1, -2)) * scale
    hidden = s["hidden"]
    if s["lengths"] is not None:
        hidden = torch.arange(Tk, device=q.device)[None, :] >= s["lengths"][:, None]
    if hidden is not None:
        scores = scores.masked_fill(hidden[:, None, None, :], -math.inf)
    p = _softmax(scores)
    out = torch.matmul(p, v)
    if not c["train"]:
        return {"out": back(out).reshape(M * G, Tq, -1)}
    do = rows(s["dout"].view(M * G, Tq, Hk * rep, D))
    dv = torch.matmul(p.transpose(-1, -2), do)
    ds = p * (torch.matmul(do, v.transpose(-1, -2)) - (do * out).sum(-1, keepdim=True)) * scale
    dq, dk = torch.matmul(ds, k), torch.matmul(ds.transpose(-1, -2), q)
    return {"out": back(out).reshape(M * G, Tq, -1), "dq": back(dq), "dk": dk.transpose(1, 2).to(dt), "dv": dv.transpose(1, 2).to(dt)}


def _plain_prefix(s):
    c = s["case"]
    P, G, Tq, Hk, D = c["prompts"], c["group"], c["tq"], c["kv_heads"], c["dim"]
    B, rep, scale, dev = P * G, c["heads"] // Hk, 1.0 / math.sqrt(D), s["q"].device
    q = s["q"].float().view(P, G, Tq, Hk, rep, D)
    kp, vp, k, v = s["kp"].float(), s["vp"].float(), s["k"].float().view(P, G, -1, Hk, D), s["v"].float().view(P, G, -1, Hk, D)
    a = torch.einsum("pgthrd,pshd->pghrts", q, kp) * scale
    b = torch.einsum("pgthrd,pgshd->pghrts", q, k) * scale
    a = a.masked_fill((torch.arange(kp.shape[1], device=dev)[None, :] >= s["prefix_lengths"][:, None])[:, None, None, None, None, :], -math.inf)
    # new token t is position lengths - Tq + t of its row's own keys and sees those up to itself
    last = s["lengths"][:, None] - Tq + torch.arange(Tq, device=dev)[None, :]
    later = torch.arange(k.shape[2], device=dev)[None, None, :] > last[:, :, None]
    b = b.masked_fill(later.view(P, G, 1, 1, Tq, -1), -math.inf)
    w = _softmax(torch.cat([a, b], -1))
    n = kp.shape[1]
    out = torch.einsum("pghrts,pshd->pgthrd", w[..., :n], vp) + torch.einsum("pghrts,pgshd->pgthrd", w[..., n:], v)
    return {"out": out.reshape(B, Tq, -1).to(s["q"].dtype)}


def _plain_rows(s):
    """Log-probability of every target (64 bits, zero where masked) and the softmax weights."""
    x = s["logits"].float()
    m = x.amax(-1, keepdim=True)
    e = torch.exp(x - m)
    total = e.sum(-1, keepdim=True, dtype=torch.float64)
    logp = x.gather(-1, s["targets"].unsqueeze(-1)).double() - m.double() - total.log()
    return logp.squeeze(-1) * s["mask"].unsqueeze(-1), e / total.float()


def _plain_grad(s, weights, slope):
    slope = slope * s["grad"]
    d = weights * (-slope).unsqueeze(-1)
    d.scatter_add_(-1, s["targets"].unsqueeze(-1), slope.unsqueeze(-1))
    return d.to(s["logits"].dtype)


def _plain_policy(s):
    c = s["case"]
    logp, weights = _plain_rows(s)
    mask = s["mask"].unsqueeze(-1).expand_as(logp).double()
    count = mask.sum()
    ratio, adv = torch.exp(logp - s["old"].double()), s["advantages"].double()[:, None, None]
    plain, clipped = ratio * adv, ratio.clamp(1 - CLIP, 1 + CLIP) * adv
    term, slope = -torch.minimum(plain, clipped), torch.where(plain <= clipped, -plain, torch.zeros_like(plain))
    if c["kl"]:
        d = s["ref"].double() - logp
        term, slope = term + KL_BETA * (torch.exp(d) - d - 1), slope + KL_BETA * (1 - torch.exp(d))
    loss = (term * mask).sum() / count
    return {"loss": loss.float(), "logp": logp.float(), "dlogits": _plain_grad(s, weights, (slope * mask / count).float())}


def _plain_preference(s):
    c = s["case"]
    n = c["pairs"]
    logp, weights = _plain_rows(s)
    mask = s["mask"].unsqueeze(-1)
    ratio = ((logp - s["ref"].double()) * mask).sum((1, 2))
    margin = ratio[:n] - ratio[n:]
    if c["loss"] == "dpo":
        x = BETA * margin
        loss, slope = torch.log1p(torch.exp(-x.abs())) + (-x).clamp(min=0), -BETA / (1 + torch.exp(x))
    elif c["loss"] == "ipo":
        d = margin - 1 / (2 * BETA)
        loss, slope = d * d, 2 * d
    else:
        d = BETA * margin - s["gap"].double()
        loss, slope = d * d, 2 * BETA * d
    slope = torch.cat([slope, -slope]) / n
    return {"loss": loss.mean().float(), "rewards": (BETA * ratio).float(),
            "dlogits": _plain_grad(s, weights, (slope[:, None, None] * mask).float().expand_as(s["ref"]))}


# ------------------------------------------------------------------------------------------------ the framework's calls
def _own(s):
    from speech_b200 import ops

    c = s["case"]
    if c["op"] == "cross":
        if not c["train"]:
            return {"out": ops.cross_attention(s["q"], s["k"], s["v"], key_lengths=s["lengths"], key_mask=s["hidden"])}
        q, k, v = (s[n].detach().requires_grad_() for n in ("q", "k", "v"))
        out = ops.cross_attention(q, k, v, key_lengths=s["lengths"], key_mask=s["hidden"])
        dq, dk, dv = torch.autograd.grad(out, (q, k, v), s["dout"])
        return {"out": out.detach(), "dq": dq, "dk": dk, "dv": dv}
    if c["op"] == "prefix":
        return {"out": ops.shared_prefix_attention(s["q"], s["kp"], s["vp"], s["k"], s["v"], s["lengths"], prefix_lengths=s["prefix_lengths"])}
    logits = s["logits"].detach().requires_grad_()
    if c["op"] == "policy":
        loss, logp = ops.policy_loss(logits, s["targets"], s["mask"], s["old"], s["advantages"], ref_logp=s["ref"], clip=CLIP,
                                     kl_beta=KL_BETA if c["kl"] else 0.0)
        return {"loss": loss.detach(), "logp": logp, "dlogits": torch.autograd.grad(loss, logits, s["grad"])[0]}
    loss, rewards = ops.preference_loss(logits, s["targets"], s["mask"], s["ref"], beta=BETA, loss_type=c["loss"], reward_gap=s["gap"])
    return {"loss": loss.detach(), "rewards": rewards, "dlogits": torch.autograd.grad(loss, logits, s["grad"])[0]}


def run(state):
    if own:
        return _own(state)
    op = state["case"]["op"]
    return {"cross": _plain_cross, "prefix": _plain_prefix, "policy": _plain_policy, "preference": _plain_preference}[op](state)


# ------------------------------------------------------------------------------------------------ what a pass cannot do without
def work(case):
    c = case
    size = {"bf16": 2, "fp16": 2, "fp32": 4}[c["dtype"]]
    if c["op"] == "cross":
        B, H, Hk, D = c["memories"] * c["group"], c["heads"], c["kv_heads"], c["dim"]
        keys = sum(_key_lengths(c)) * (0.7 if c["hidden"] == "mask" else 1.0)
        if c["hidden"] == "mask" and c["memories"] > 2:
            keys = keys * (c["memories"] - 1) / c["memories"]
        qo, kv = B * c["tq"] * H * D * size, keys * Hk * D * size
        products = 2.0 * c["group"] * c["tq"] * H * D * keys
        if not c["train"]:
            return {"bytes": 2 * qo + 2 * kv, "flops": 2 * products}
        # forward reads q, k, v and writes out; backward reads dout besides and writes dq and all of dk and dv
        return {"bytes": 4 * qo + 2 * kv + 2 * c["memories"] * c["tk"] * Hk * D * size, "flops": 7 * products}
    if c["op"] == "prefix":
        B, H, Hk, D = c["prompts"] * c["group"], c["heads"], c["kv_heads"], c["dim"]
        prefix, mine = sum(_prefix_lengths(c)), sum(_own_lengths(c))
        return {"bytes": 2 * (prefix + mine) * Hk * D * size + 2 * B * c["tq"] * H * D * size,
                "flops": 4.0 * c["tq"] * H * D * (prefix * c["group"] + mine)}
    n, steps = _steps(c)
    rows, all_rows = sum(steps) * c["books"], n * c["steps"] * c["books"]
    per_row = {"policy": 8 + 4 + 4 + (4 if c.get("kl") else 0), "preference": 8 + 4}[c["op"]]
    # masked rows are not read, but their gradient is written
    return {"bytes": rows * c["vocab"] * size + all_rows * c["vocab"] * size + rows * per_row, "flops": 6.0 * rows * c["vocab"]}


# ------------------------------------------------------------------------------------------------ in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "cross":
        H, Hk, G = case["heads"], case["kv_heads"], case["group"]
        q, k, v = (s[n].double().requires_grad_(case["train"]) for n in ("q", "k", "v"))
        outs = []
        for m in range(case["memories"]):
            seen = torch.ones(case["tk"], dtype=torch.bool, device=q.device)
            if s["hidden"] is not None:
                seen = ~s["hidden"][m]
            if s["lengths"] is not None:
                seen = torch.arange(case["tk"], device=q.device) < s["lengths"][m]
            km, vm = (x[m][seen].repeat_interleave(H // Hk, dim=1) for x in (k, v))         # [keys, H, D]
            sc = torch.einsum("gthd,shd->ghts", q[m * G:(m + 1) * G], km) / math.sqrt(case["dim"])
            outs.append(torch.einsum("ghts,shd->gthd", torch.softmax(sc, -1), vm))
        out = torch.cat(outs).flatten(2)
        if not case["train"]:
            return {"out": out}
        dq, dk, dv = torch.autograd.grad(out, (q, k, v), s["dout"].double())
        return {"out": out.detach(), "dq": dq, "dk": dk, "dv": dv}
    if case["op"] == "prefix":
        G, Tq, rep = case["group"], case["tq"], case["heads"] // case["kv_heads"]
        q, outs = s["q"].double(), []
        for b in range(q.shape[0]):
            n, mine = int(s["prefix_lengths"][b // G]), int(s["lengths"][b])
            kb, vb = (torch.cat([x[b // G, :n], y[b, :mine]]).double().repeat_interleave(rep, dim=1) for x, y in ((s["kp"], s["k"]), (s["vp"], s["v"])))
            rows = []
            for t in range(Tq):
                upto = n + max(0, mine - Tq + 1 + t)
                w = torch.softmax(torch.einsum("hd,shd->hs", q[b, t], kb[:upto]) / math.sqrt(case["dim"]), -1)
                rows.append(torch.einsum("hs,shd->hd", w, vb[:upto]).flatten())
            outs.append(torch.stack(rows))
        return {"out": torch.stack(outs)}
    logits, n = s["logits"], s["logits"].shape[0]
    picked = [torch.log_softmax(logits[i].double(), -1).gather(-1, s["targets"][i].unsqueeze(-1)).squeeze(-1) for i in range(n)]
    logp = torch.where(s["mask"].unsqueeze(-1), torch.stack(picked), 0.0).requires_grad_()
    if case["op"] == "policy":
        ratio, adv = (logp - s["old"].double()).exp(), s["advantages"].double().view(-1, 1, 1)
        term = -torch.min(ratio * adv, ratio.clamp(1 - CLIP, 1 + CLIP) * adv)
        if case["kl"]:
            d = s["ref"].double() - logp
            term = term + KL_BETA * (d.exp() - 1 - d)
        loss = term[s["mask"].unsqueeze(-1).expand_as(term)].mean()
        second = {"logp": logp.detach()}
    else:
        pairs = n // 2
        ratio = ((logp - s["ref"].double()) * s["mask"].unsqueeze(-1)).sum((1, 2))
        margin = ratio[:pairs] - ratio[pairs:]
        loss = {"dpo": lambda: -torch.nn.functional.logsigmoid(BETA * margin), "ipo": lambda: (margin - 0.5 / BETA) ** 2,
                "rpo_sq": lambda: (BETA * margin - s["gap"].double()) ** 2}[case["loss"]]().mean()
        second = {"rewards": (BETA * ratio).detach()}
    (slope,) = torch.autograd.grad(loss, logp, s["grad"].double())
    slope = slope * s["mask"].unsqueeze(-1)
    grads = torch.empty(logits.shape, dtype=torch.float64, device=logits.device)
    for i in range(n):
        grads[i] = -slope[i].unsqueeze(-1) * torch.softmax(logits[i].double(), -1)
        grads[i].scatter_add_(-1, s["targets"][i].unsqueeze(-1), slope[i].unsqueeze(-1))
    return {"loss": loss.detach(), **second, "dlogits": grads}
