"""The vocabulary losses written out in 64 bits, from the formulas alone, with
the gradient of the logits, and how far an fp32 computation may be off them."""
from __future__ import annotations

import math

import torch


def logp64(logits, ids, t):
    """log-probabilities [rows, k] and the rows' probabilities [rows, vocab]."""
    z = logits.double() / t
    m = z.amax(1, keepdim=True)
    e = (z - m).exp()
    s = e.sum(1, keepdim=True)
    return (z - m).gather(1, ids) - s.log(), e / s


def policy(logits, y, old, adv, ref, w, lo, hi, beta, t, denom):
    n, v = logits.shape
    counted = y >= 0 if w is None else (y >= 0) & (w != 0)
    w = torch.where(y >= 0, torch.ones_like(old).double() if w is None else w.double(), 0.0)
    denom = float(w.sum()) if denom is None else denom
    lp, p = logp64(logits, y.clamp(min=0)[:, None], t)
    lp = lp[:, 0]
    r, a = (lp - old.double()).exp(), adv.double()
    stopped = ((a > 0) & (r > 1 + hi)) | ((a < 0) & (r < 1 - lo))
    each = -torch.minimum(r * a, r.clamp(1 - lo, 1 + hi) * a)
    slope = torch.where(stopped, 0.0, -a * r)
    bend = torch.where(stopped, 0.0, (a * r).abs())  # of the slope, in logp
    kl = None
    if ref is not None:
        d = ref.double() - lp
        kl = torch.where(counted, d.exp() - d - 1, 0.0)
        each = each + beta * (d.exp() - d - 1)
        slope = slope + beta * (1 - d.exp())
        bend = bend + beta * d.exp()
    scale = w / denom if denom > 0 else torch.zeros_like(w)
    loss = torch.where(counted, each * scale, 0.0).sum()
    slope, bend = (torch.where(counted, x * scale, 0.0) / t for x in (slope, bend))
    g = -p
    g[torch.arange(n, device=g.device), y.clamp(min=0)] += 1
    g = torch.where(counted[:, None], g * slope[:, None], 0.0)
    return {"loss": loss, "logp": torch.where(counted, lp, 0.0), "kl": kl, "clipped": stopped & counted, "grad": g,
            "p": p, "slope": slope, "bend": bend, "scale": scale, "each": torch.where(counted, each, 0.0)}


def distill(logits, ids, teacher, w, t, denom):
    n, v = logits.shape
    w = torch.ones(n, device=logits.device, dtype=torch.float64) if w is None else w.double()
    there = ids >= 0
    tz = torch.where(there, teacher.double() / t, -math.inf)
    tz = torch.where(there.any(1, keepdim=True), tz, 0.0)
    q = torch.where(there, tz.softmax(1), 0.0)
    lp, p = logp64(logits, ids.clamp(min=0), t)
    kl = torch.where(q > 0, q * (q.log() - lp), 0.0).sum(1)
    kl = torch.where(w != 0, kl, 0.0)
    denom = float(w.sum()) if denom is None else denom
    scale = w / denom if denom > 0 else torch.zeros_like(w)
    target = torch.zeros_like(p).scatter_add_(1, ids.clamp(min=0), q)
    slope = -scale * q.sum(1) / t
    g = torch.where((slope != 0)[:, None], -slope[:, None] * (p * q.sum(1, keepdim=True) - target), 0.0)
    return {"loss": (kl * scale).sum(), "kl": kl, "grad": g, "p": p, "slope": slope, "scale": scale}


def preference(logits, y, ref, ends, beta, eps, normalized, t):
    n, v = logits.shape
    counted = y >= 0
    lp, p = logp64(logits, y.clamp(min=0)[:, None], t)
    lp = torch.where(counted, lp[:, 0], 0.0)
    k = (len(ends) - 1) // 2
    per = [1.0 / max(1, int(counted[a:b].sum())) if normalized else 1.0 for a, b in zip(ends, ends[1:])]
    s = torch.stack([lp[a:b].sum() * f for (a, b), f in zip(zip(ends, ends[1:]), per)])
    r = beta * (s - (0 if ref is None else ref.double()))
    h = r[:k] - r[k:]
    loss = ((1 - eps) * (1 + (-h).exp()).log() + eps * (1 + h.exp()).log()).mean()
    dh = (-(1 - eps) / (1 + h.exp()) + eps / (1 + (-h).exp())) * beta / k
    slope = torch.zeros(n, dtype=torch.float64, device=logits.device)
    for i, (a, b) in enumerate(zip(ends, ends[1:])):
        slope[a:b] = dh[i % k] * (1 if i < k else -1) * per[i]
    slope = torch.where(counted, slope, 0.0) / t
    g = -p
    g[torch.arange(n, device=g.device), y.clamp(min=0)] += 1
    return {"loss": loss, "rewards": r, "grad": g * slope[:, None], "p": p, "slope": slope, "h": h, "dh": dh, "logp": lp}


def logp_off(logits, t, logp):
    """How far a log-probability may be off (2^-24 is half a step of fp32 at 1).
    A thread adds at most vocab / 256 terms to its sum and 64 more to join the
    threads, each addition off by half a step; a term is off by 2^-22 (the
    exponential's two steps) and by half a step of its exponent, which weighs
    at most 1; the scale log2(e) / T is off by half a step, which moves the
    log-probability by that share of the logits' spread, at most 2 max |z|;
    and the result is rounded."""
    z = logits.double().abs() / t
    z = torch.where(z < 1e6, z, 0.0).amax(1)  # beyond that entries are masked, or a row's own base is taken off first
    return 2.0 ** -24 * (logits.shape[1] / 256 + 64 + 4 + 1 + 2 * z * 1.45 + logp.abs())


def grad_off(ref, dtype, off, slope_off):
    """How far a gradient may be off: half a step of its type, what the
    probability carries over from the row's sum (`off`) and its own exponential
    (2^-22, and half a step of an exponent), and the slope's error (per row).
    Where 1 - p is taken the probability's error counts against 1."""
    half = torch.finfo(dtype).eps / 2
    p = ref["p"]
    p_off = p * (off[:, None] + 2.0 ** -21 + 2.0 ** -23 * (-p.clamp(min=1e-300).log2()))
    d = ref["slope"].abs()[:, None] * p_off + slope_off[:, None] * (ref["grad"] / torch.where(
        ref["slope"] == 0, 1.0, ref["slope"])[:, None]).abs() + 2.0 ** -22 * ref["grad"].abs()
    # below the types' normal range: half a step of a subnormal, and exponentials under 2^-126 are zero.
    # They count from an integer that is at most 1/2 above the row's maximum, so the sum that divides
    # them is at least 2^-1/2 and what is lost at most 2^-125.5 of the slope
    low = torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps + 2.0 ** -125.5 * ref["slope"].abs()[:, None]
    return d * (1 + half) + half * ref["grad"].abs() + low
