"""The vocabulary losses (token log-probabilities, clipped policy loss, preference loss, distillation from a
teacher's top logits) on sizes of real use, in their plain form and through the package's entry points.

A case names an operator (``op``), the logits' type, the number of token rows, the vocabulary and what the
operator needs besides; ``run`` computes the operator's outputs and, where ``train`` is true, the gradient
of the logits.
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def listed():
    return [
        # one sampled token scored by an inference rank: launch latency and one 303 KB row
        {"name": "logprobs-1-token", "op": "logprobs", "dtype": "bf16", "rows": 1, "vocab": 151552, "train": False},
        # old / reference log-probabilities of a rollout batch before a policy step (GLM-4-9B vocabulary)
        {"name": "logprobs-rollout", "op": "logprobs", "dtype": "bf16", "rows": 4096, "vocab": 151552, "train": False},
        # a user's own loss on top of the log-probabilities, fp32 logits: forward and backward
        {"name": "logprobs-train-fp32", "op": "logprobs", "dtype": "fp32", "rows": 777, "vocab": 151936, "train": True},
        # a policy step's micro batch of 8192 tokens, KL to a reference model, part of the tokens is prompt
        {"name": "policy-8192", "op": "policy", "dtype": "bf16", "rows": 8192, "vocab": 151552, "train": True,
         "kl": 0.05, "masked": 0.1, "temperature": 1.0},
        # a chunk of the output head in fp32 (Qwen3.5-35B-A3B vocabulary), no KL term, sampling temperature 0.7
        {"name": "policy-fp32", "op": "policy", "dtype": "fp32", "rows": 1024, "vocab": 151936, "train": True,
         "kl": 0.0, "masked": 0.0, "temperature": 0.7},
        # an odd vocabulary in fp16: no row but the first starts on a 16-byte border
        {"name": "policy-odd-fp16", "op": "policy", "dtype": "fp16", "rows": 515, "vocab": 32003, "train": True,
         "kl": 0.02, "masked": 0.25, "temperature": 1.0},
        # the example's small model: launch latency
        {"name": "policy-small", "op": "policy", "dtype": "bf16", "rows": 16, "vocab": 1000, "train": True,
         "kl": 0.05, "masked": 0.0, "temperature": 1.0},
        # 8 chosen and 8 rejected answers of one padded length
        {"name": "preference-16x256", "op": "preference", "dtype": "bf16", "pairs": 8, "length": 256, "ragged": False,
         "vocab": 151936, "smoothing": 0.0, "normalized": False, "train": True},
        # packed answers of uneven lengths, mean log-probability, label smoothing
        {"name": "preference-packed", "op": "preference", "dtype": "fp32", "pairs": 5, "length": 61, "ragged": True,
         "vocab": 32000, "smoothing": 0.1, "normalized": True, "train": True},
        # distillation on the teacher's 64 best tokens
        {"name": "distill-4096-top64", "op": "distill", "dtype": "bf16", "rows": 4096, "vocab": 151552, "top": 64,
         "train": True, "masked": 0.05, "temperature": 1.0},
        # a short sequence against 128 entries at temperature 2
        {"name": "distill-33-top128", "op": "distill", "dtype": "bf16", "rows": 33, "vocab": 151936, "top": 128,
         "train": True, "masked": 0.0, "temperature": 2.0},
        # fp32 logits of an odd vocabulary, 20 entries as a log of top log-probabilities holds
        {"name": "distill-odd-fp32", "op": "distill", "dtype": "fp32", "rows": 600, "vocab": 50021, "top": 20,
         "train": True, "masked": 0.1, "temperature": 1.0},
    ]


def draw(rng):
    def log_int(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    size = 4 if dtype == "fp32" else 2
    vocab = log_int(1000, 152000)
    if rng.random() < 0.5:
        vocab = max(1000, vocab // 64 * 64)
    most = max(1, min(8192, 8192 * 151552 * 2 // (vocab * size)))
    op = rng.choice(["logprobs", "policy", "policy", "preference", "distill"])
    case = {"op": op, "dtype": dtype, "vocab": vocab, "train": True}
    if op == "preference":
        case["pairs"] = log_int(1, 16)
        case["length"] = max(1, min(log_int(4, 512), most // (2 * case["pairs"])))
        case["ragged"] = rng.random() < 0.5
        case["smoothing"] = rng.choice([0.0, 0.1])
        case["normalized"] = rng.random() < 0.5
        return case
    case["rows"] = log_int(1, most)
    if op == "logprobs":
        case["train"] = rng.random() < 0.5
        return case
    case["masked"] = rng.choice([0.0, 0.1, 0.3])
    case["temperature"] = rng.choice([0.7, 1.0, 2.0])
    if op == "policy":
        case["kl"] = rng.choice([0.0, 0.02, 0.1])
    else:
        case["top"] = log_int(1, 128)
    return case


CLIP_LOW, CLIP_HIGH, BETA = 0.2, 0.28, 0.1


def _rows(case):
    return 2 * case["pairs"] * case["length"] if case["op"] == "preference" else case["rows"]


def _logp64(logits, tokens, temperature):
    """log-probability of each token in 64 bits, a few rows at a time."""
    out = []
    for x, y in zip(logits.split(256), tokens.split(256)):
        z = x.double() / temperature
        out.append(z.gather(1, y.clamp(min=0)[:, None])[:, 0] - z.logsumexp(1))
    return torch.cat(out)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    n, v, t = _rows(case), case["vocab"], case.get("temperature", 1.0)
    # logits of a language model: wide, and the last columns of the head are padding of the vocabulary
    logits = torch.randn(n, v, device="cuda", generator=g, dtype=DTYPES[case["dtype"]]).mul_(2.5)
    logits[:, v - v // 500:] = -math.inf
    # tokens sampled from the model
    tokens = torch.cat([(x.float() / t - torch.rand(x.shape, device="cuda", generator=g).log_().neg_().log_()).argmax(1)
                        for x in logits.split(256)])
    state = {"case": case, "logits": logits, "tokens": tokens}

    def noise(k, scale):
        return torch.randn(k, device="cuda", generator=g, dtype=torch.float64) * scale

    if case["op"] == "logprobs":
        tokens[torch.rand(n, device="cuda", generator=g) < 0.1] = -100  # prompt tokens, not scored
        state["upstream"] = noise(n, 1.0 / n).float()
    elif case["op"] == "policy":
        logp = _logp64(logits, tokens, t)
        d = noise(n, 0.2)  # how far the policy has moved; a ratio at the clip's very border has no one gradient
        for edge in (math.log(1 - CLIP_LOW), math.log(1 + CLIP_HIGH)):
            d = torch.where((d - edge).abs() < 1e-3, d + 4e-3, d)
        state["old"] = (logp - d).float()
        state["ref"] = (logp + noise(n, 0.3)).float() if case["kl"] else None
        state["advantages"] = noise(n, 1.0).float()
        state["weights"] = (torch.rand(n, device="cuda", generator=g) >= case["masked"]).float()
        state["weights"][0] = 1.0
    elif case["op"] == "preference":
        s = 2 * case["pairs"]
        total = s * case["length"]
        if case["ragged"]:  # sequences of uneven lengths, one after another
            cuts = torch.rand(s - 1, device="cuda", generator=g).mul_(total).long().sort().values
            ends = torch.tensor([total], device="cuda")
            state["cu_seqlens"] = torch.cat([torch.zeros_like(ends), cuts, ends]).int()
        else:  # prompts in front and padding behind are not scored
            length = case["length"]
            first = torch.randint(0, length // 2 + 1, (s, 1), device="cuda", generator=g)
            last = torch.randint(length // 2, length + 1, (s, 1), device="cuda", generator=g)
            at = torch.arange(length, device="cuda")
            tokens[((at < first) | (at >= last)).view(-1)] = -100
            state["cu_seqlens"] = None
        offsets = _offsets(state)
        logp = torch.where(tokens >= 0, _logp64(logits, tokens, 1.0), 0.0)
        sums = torch.cat([torch.zeros(1, device="cuda", dtype=torch.float64), logp.cumsum(0)])[offsets]
        sums = sums[1:] - sums[:-1]
        if case["normalized"]:
            sums = sums / _counts(state).clamp(min=1)
        state["ref"] = (sums + noise(s, 0.3 if case["normalized"] else 3.0)).float()
    else:
        k = case["top"]
        best = [(x.float() + torch.randn(x.shape, device="cuda", generator=g)).topk(k, 1) for x in logits.split(256)]
        state["ids"] = torch.cat([b.indices for b in best])
        state["teacher"] = torch.cat([b.values for b in best]).to(DTYPES[case["dtype"]])
        if k > 4:  # some lists are shorter: the rest is padding
            short = torch.rand(n, device="cuda", generator=g) < 0.2
            state["ids"][:, -2:] = torch.where(short[:, None], -1, state["ids"][:, -2:])
        state["weights"] = (torch.rand(n, device="cuda", generator=g) >= case["masked"]).float()
        state["weights"][0] = 1.0
    if case["train"]:
        state["logits"].requires_grad_(True)
    return state


def _offsets(state):
    case = state["case"]
    if state["cu_seqlens"] is not None:
        return state["cu_seqlens"].long()
    return torch.arange(2 * case["pairs"] + 1, device="cuda") * case["length"]


def _counts(state):
    offsets = _offsets(state)
    c = (state["tokens"] >= 0).long().cumsum(0)
    c = torch.cat([torch.zeros(1, dtype=torch.long, device="cuda"), c])[offsets]
    return c[1:] - c[:-1]


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ---- the package's entry points -------------------------------------------------------------------------


def _run_own(state):
    import results_b200 as lz

    case, logits = state["case"], state["logits"]
    if case["op"] == "logprobs":
        logp = lz.token_logprobs(logits, state["tokens"])
        if not case["train"]:
            return {"logp": logp}
        grad, = torch.autograd.grad(logp, logits, state["upstream"])
        return {"logp": logp.detach(), "grad": grad}
    if case["op"] == "policy":
        out = lz.policy_loss(logits, state["tokens"], state["old"], state["advantages"], ref_logp=state["ref"],
                             weights=state["weights"], clip_low=CLIP_LOW, clip_high=CLIP_HIGH, kl_coef=case["kl"],
                             temperature=case["temperature"])
        grad, = torch.autograd.grad(out.loss, logits)
        res = {"loss": out.loss.detach(), "logp": out.logp, "clipped": out.clipped, "grad": grad}
        if case["kl"]:
            res["kl"] = out.kl
        return res
    if case["op"] == "preference":
        x, y = logits, state["tokens"]
        if state["cu_seqlens"] is None:
            x, y = x.view(-1, case["length"], case["vocab"]), y.view(-1, case["length"])
        out = lz.preference_loss(x, y, ref_logp=state["ref"], cu_seqlens=state["cu_seqlens"], beta=BETA,
                                 label_smoothing=case["smoothing"], length_normalized=case["normalized"])
        grad, = torch.autograd.grad(out.loss, logits)
        return {"loss": out.loss.detach(), "chosen": out.chosen_rewards, "rejected": out.rejected_rewards, "grad": grad}
    out = lz.distill_loss(logits, state["ids"], state["teacher"], weights=state["weights"],
                          temperature=case["temperature"])
    grad, = torch.autograd.grad(out.loss, logits)
    return {"loss": out.loss.detach(), "kl": out.kl, "grad": grad}


# ---- the plain form ----------------------------------------------------------------------------------------


def _softmax_parts(z):
    m = z.amax(1, keepdim=True)
    return m + (z - m).exp().sum(1, keepdim=True).log()


def _spread(z, lse, y, coef, dtype):
    """coef_r * ([j = y_r] - p_rj), rounded once."""
    grad = (z - lse).exp() * -coef[:, None]
    grad.scatter_add_(1, y[:, None], coef[:, None])
    return grad.to(dtype)


@torch.no_grad()
def _run_plain(state):
    case, logits = state["case"], state["logits"]
    t = case.get("temperature", 1.0)
    z = logits.float()
    if t != 1.0:
        z = z / t
    lse = _softmax_parts(z)
    if case["op"] == "distill":
        return _plain_distill(state, z, lse, t)
    counted = state["tokens"] >= 0
    y = state["tokens"].clamp(min=0)
    logp = z.gather(1, y[:, None])[:, 0] - lse[:, 0]
    logp = torch.where(counted, logp, 0.0)
    if case["op"] == "logprobs":
        if not case["train"]:
            return {"logp": logp}
        coef = torch.where(counted, state["upstream"], 0.0)
        return {"logp": logp, "grad": _spread(z, lse, y, coef, logits.dtype)}
    if case["op"] == "policy":
        w, a = state["weights"], state["advantages"]
        counted = counted & (w != 0)
        logp = torch.where(counted, logp, 0.0)
        ratio = (logp - state["old"]).exp()
        surrogate = torch.minimum(ratio * a, ratio.clamp(1 - CLIP_LOW, 1 + CLIP_HIGH) * a)
        clipped = (((a > 0) & (ratio > 1 + CLIP_HIGH)) | ((a < 0) & (ratio < 1 - CLIP_LOW))) & counted
        each = -surrogate
        slope = torch.where(clipped, 0.0, -a * ratio)
        kl = None
        if case["kl"]:
            d = torch.where(counted, state["ref"] - logp, 0.0)
            kl = d.expm1() - d
            each = each + case["kl"] * kl
            slope = slope - case["kl"] * d.expm1()
        scale = w / w.sum()
        loss = torch.where(counted, each * scale, 0.0).sum()
        coef = torch.where(counted, slope * scale, 0.0)
        res = {"loss": loss, "logp": logp, "clipped": clipped, "grad": _spread(z, lse, y, coef / t, logits.dtype)}
        if kl is not None:
            res["kl"] = kl
        return res
    # preference: sums in 64 bits, since differences of long sums are what counts
    offsets = _offsets(state)
    sums = torch.cat([torch.zeros(1, dtype=torch.float64, device="cuda"), logp.double().cumsum(0)])[offsets]
    sums = sums[1:] - sums[:-1]
    per = torch.ones_like(sums)
    if case["normalized"]:
        per = 1.0 / _counts(state).clamp(min=1)
        sums = sums * per
    rewards = BETA * (sums - state["ref"].double())
    p, eps = case["pairs"], case["smoothing"]
    h = rewards[:p] - rewards[p:]
    soft = torch.log1p(torch.exp(-h.abs()))
    loss = ((1 - eps) * (soft + (-h).clamp(min=0)) + eps * (soft + h.clamp(min=0))).mean()
    dh = (eps / (1 + torch.exp(-h)) - (1 - eps) / (1 + torch.exp(h))) * BETA / p
    each = torch.cat([dh, -dh]) * per
    row = torch.arange(logp.numel(), device="cuda")
    seq = torch.searchsorted(offsets[1:].contiguous(), row, right=True)
    coef = torch.where(counted, each[seq], 0.0).float()
    return {"loss": loss.float(), "chosen": rewards[:p].float(), "rejected": rewards[p:].float(),
            "grad": _spread(z, lse, y, coef, logits.dtype)}


def _plain_distill(state, z, lse, t):
    ids, w = state["ids"], state["weights"]
    there = ids >= 0
    teacher = torch.where(there, state["teacher"].float() / t, -math.inf)
    m = teacher.amax(1, keepdim=True)
    e = (teacher - m).exp()
    s = e.sum(1, keepdim=True)
    q = e / s
    logq = teacher - m - s.log()
    at = ids.clamp(min=0)
    student = z.gather(1, at) - lse
    kl = torch.where(there & (q > 0), q * (logq - student), 0.0).sum(1)
    kl = torch.where(w != 0, kl, 0.0)
    scale = w / w.sum()
    grad = (z - lse).exp() * (scale / t)[:, None]
    grad.scatter_add_(1, at, -q * (scale / t)[:, None])
    return {"loss": (kl * scale).sum(), "kl": kl, "grad": grad.to(state["logits"].dtype)}


# ---- what a pass cannot do without ------------------------------------------------------------------------


def work(case):
    n, v, size = _rows(case), case["vocab"], 4 if case["dtype"] == "fp32" else 2
    once = n * v * size
    small = n * 4 * {"logprobs": 3, "policy": 8, "preference": 2, "distill": 3}[case["op"]]
    if case["op"] == "distill":
        small += n * case["top"] * (8 + size)
    if not case["train"]:
        return {"bytes": once + small, "flops": 4 * n * v}
    return {"bytes": 2 * once + small, "flops": 7 * n * v}


# ---- the definitions in 64 bits ------------------------------------------------------------------------------


@torch.no_grad()
def exact(case, seed):
    state = prepare(case, seed)
    x, t = state["logits"].detach(), case.get("temperature", 1.0)
    n = x.shape[0]
    parts = [slice(i, min(i + 256, n)) for i in range(0, n, 256)]
    if case["op"] == "distill":
        return _exact_distill(state, x, t, parts)
    y = state["tokens"]
    ok = y >= 0
    if case["op"] == "policy":
        ok = ok & (state["weights"] != 0)
    logp = torch.cat([torch.log_softmax(x[s].double() / t, 1).gather(1, y[s].clamp(min=0)[:, None]) for s in parts])[:, 0]
    logp = logp.masked_fill(~ok, 0.0)
    res = {"logp": logp}
    if case["op"] == "logprobs":
        slope = state["upstream"].double()
    elif case["op"] == "policy":
        w = state["weights"].double()
        share = w / w.sum()
        a, r = state["advantages"].double(), torch.exp(logp - state["old"].double())
        low, high = 1.0 - CLIP_LOW, 1.0 + CLIP_HIGH
        stopped = torch.where(a > 0, r > high, (r < low) & (a < 0)) & ok
        gain = torch.where(stopped, torch.where(a > 0, a * high, a * low), a * r)
        each, slope = -gain, torch.where(stopped, 0.0, -a * r)
        if case["kl"]:
            d = (state["ref"].double() - logp).masked_fill(~ok, 0.0)
            res["kl"] = torch.expm1(d) - d
            each, slope = each + case["kl"] * res["kl"], slope + case["kl"] * (1.0 - torch.exp(d))
        res["loss"] = (each * share).masked_fill(~ok, 0.0).sum()
        slope = slope * share
        res["clipped"] = None
    else:
        ends = _offsets(state).tolist()
        p = case["pairs"]
        total = torch.stack([logp[a:b].sum() for a, b in zip(ends, ends[1:])])
        length = torch.tensor([max(1, int(ok[a:b].sum())) if case["normalized"] else 1 for a, b in zip(ends, ends[1:])],
                              device="cuda")
        reward = BETA * (total / length - state["ref"].double())
        h = reward[:p] - reward[p:]
        eps = case["smoothing"]
        log_sigmoid = torch.nn.functional.logsigmoid
        dh = -(1 - eps) * torch.sigmoid(-h) + eps * torch.sigmoid(h)
        res = {"loss": (-(1 - eps) * log_sigmoid(h) - eps * log_sigmoid(-h)).mean(), "chosen": reward[:p], "rejected": reward[p:]}
        of_seq = torch.cat([dh, -dh]) * BETA / p / length
        slope = torch.cat([of_seq[i].expand(b - a) for i, (a, b) in enumerate(zip(ends, ends[1:]))])
    if case["train"]:
        slope = (slope / t).masked_fill(~ok, 0.0)
        res["grad"] = torch.empty(x.shape, dtype=torch.float64, device="cuda")
        for s in parts:
            g = torch.softmax(x[s].double() / t, 1).neg_()
            g[torch.arange(g.shape[0], device="cuda"), y[s].clamp(min=0)] += 1.0
            res["grad"][s] = g * slope[s, None]
    return res


def _exact_distill(state, x, t, parts):
    w = state["weights"].double()
    share = w / w.sum()
    grad = torch.empty(x.shape, dtype=torch.float64, device="cuda")
    kls = []
    for s in parts:
        ids, z = state["ids"][s], x[s].double() / t
        q = torch.softmax((state["teacher"][s].double() / t).masked_fill(ids < 0, -math.inf), 1)
        logp = torch.log_softmax(z, 1)
        kls.append((torch.xlogy(q, q) - torch.where(q > 0, q * logp.gather(1, ids.clamp(min=0)), 0.0)).sum(1))
        target = torch.zeros_like(z).scatter_add_(1, ids.clamp(min=0), q)
        grad[s] = (logp.exp() - target) * (share[s] / t)[:, None]
    kl = torch.cat(kls).masked_fill(w == 0, 0.0)
    return {"loss": (kl * share).sum(), "kl": kl, "grad": grad}
