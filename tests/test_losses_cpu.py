"""Vocabulary losses on CPU tensors: against the formulas in 64 bits and against
differences, rows that do not count, and every refusal (the checks are the same
for CUDA tensors)."""
import math

import pytest
import torch

import results_b200 as lz
from tests import _losses as oracle


def _g(seed):
    return torch.Generator().manual_seed(seed)


def _policy_inputs(n, v, seed, ref=True):
    g = _g(seed)
    x = torch.randn(n, v, generator=g) * 2
    y = torch.randint(0, v, (n,), generator=g)
    lp = oracle.logp64(x, y[:, None], 1.0)[0][:, 0]
    old = (lp + 0.3 * torch.randn(n, generator=g)).float()
    adv = torch.randn(n, generator=g)
    r = (lp + 0.3 * torch.randn(n, generator=g)).float() if ref else None
    return x, y, old, adv, r


# fp32 in and out of 64-bit torch operations: half a step of each rounding, and a
# few steps of the 64-bit sums, far below 2^-22 relative
REL = 2.0 ** -22


def _close(a, b, scale=None):
    b = b.double()
    s = b.abs() if scale is None else scale
    assert torch.all((a.double() - b).abs() <= REL * s + 1e-12), float(((a.double() - b).abs() - REL * s).max())


@pytest.mark.parametrize("n,v", [(1, 1), (1, 7), (9, 50), (33, 257)])
@pytest.mark.parametrize("temperature", [1.0, 0.5])
def test_token_logprobs(n, v, temperature):
    g = _g(n + v)
    x = (torch.randn(n, v, generator=g) * 3).requires_grad_(True)
    y = torch.randint(0, v, (n,), generator=g)
    y[n // 2] = -100
    up = torch.randn(n, generator=g)
    out = lz.token_logprobs(x, y, temperature=temperature)
    grad, = torch.autograd.grad(out, x, up)
    lp, p = oracle.logp64(x.detach(), y.clamp(min=0)[:, None], temperature)
    on = (y >= 0).double()
    _close(out, lp[:, 0] * on)
    want = -p
    want[torch.arange(n), y.clamp(min=0)] += 1
    slope = up.double() * on / temperature
    _close(grad, want * slope[:, None], slope.abs()[:, None].expand_as(grad))


@pytest.mark.parametrize("weighted", [False, True])
@pytest.mark.parametrize("ref", [False, True])
def test_policy_loss(weighted, ref):
    x, y, old, adv, r = _policy_inputs(40, 60, 3, ref)
    y[5] = -100
    w = torch.rand(40, generator=_g(9)) if weighted else None
    if weighted:
        w[7] = 0
    x.requires_grad_(True)
    out = lz.policy_loss(x, y, old, adv, ref_logp=r, weights=w, clip_low=0.2, clip_high=0.25,
                         kl_coef=0.1 if ref else 0.0)
    grad, = torch.autograd.grad(out.loss, x)
    want = oracle.policy(x.detach(), y, old, adv, r, w, 0.2, 0.25, 0.1 if ref else 0.0, 1.0, None)
    _close(out.loss, want["loss"], (want["each"] * want["scale"]).abs().sum())
    _close(out.logp, want["logp"])
    assert torch.equal(out.clipped, want["clipped"]) and out.clipped.any() and not out.clipped.all()
    if ref:
        # the reference and the log-probabilities are differences: off by REL of what they are taken from
        _close(out.kl, want["kl"], want["kl"] + 1)
    else:
        assert out.kl is None
    _close(grad, want["grad"], want["slope"].abs()[:, None].expand_as(grad))
    assert torch.all(grad[5] == 0) and (not weighted or torch.all(grad[7] == 0))


@pytest.mark.parametrize("packed", [False, True])
@pytest.mark.parametrize("normalized", [False, True])
def test_preference_loss(packed, normalized):
    g = _g(4)
    n, v = 4 * 6, 31
    x = torch.randn(n, v, generator=g).requires_grad_(True)
    y = torch.randint(0, v, (n,), generator=g)
    y[torch.rand(n, generator=g) < 0.2] = -100
    ends = [0, 6, 12, 18, 24] if not packed else [1, 4, 4, 15, 22]  # an empty one; rows outside of all
    ref = torch.randn(4, generator=g)
    if packed:
        out = lz.preference_loss(x, y, ref_logp=ref, cu_seqlens=torch.tensor(ends), label_smoothing=0.1,
                                 length_normalized=normalized)
    else:
        out = lz.preference_loss(x.view(4, 6, v), y.view(4, 6), ref_logp=ref, label_smoothing=0.1,
                                 length_normalized=normalized)
    grad, = torch.autograd.grad(out.loss, x)
    want = oracle.preference(x.detach(), y, ref, ends, 0.1, 0.1, normalized, 1.0)
    _close(out.loss, want["loss"])
    _close(out.chosen_rewards, want["rewards"][:2], want["rewards"][:2].abs() + 1)
    _close(out.rejected_rewards, want["rewards"][2:], want["rewards"][2:].abs() + 1)
    _close(grad, want["grad"], want["slope"].abs()[:, None].expand_as(grad))
    if packed:
        assert torch.all(grad[0] == 0) and torch.all(grad[22:] == 0)


@pytest.mark.parametrize("k", [1, 5, 20])
@pytest.mark.parametrize("temperature", [1.0, 2.0])
def test_distill_loss(k, temperature):
    g = _g(k)
    n, v = 13, 40
    x = (torch.randn(n, v, generator=g) * 2).requires_grad_(True)
    ids = torch.stack([torch.randperm(v, generator=g)[:k] for _ in range(n)])
    t = torch.randn(n, k, generator=g) * 2
    ids[2] = -1          # an empty list
    if k > 3:
        ids[3, -2:] = -1     # padding
        ids[4, 1] = ids[4, 3]  # an index that stands twice
    w = torch.rand(n, generator=g)
    w[6] = 0
    out = lz.distill_loss(x, ids, t, weights=w, temperature=temperature)
    grad, = torch.autograd.grad(out.loss, x)
    want = oracle.distill(x.detach(), ids, t, w, temperature, None)
    _close(out.kl, want["kl"], want["kl"] + 1)
    _close(out.loss, want["loss"], want["loss"] + 1)
    _close(grad, want["grad"], want["slope"].abs()[:, None].expand_as(grad))
    assert torch.all(grad[2] == 0) and torch.all(grad[6] == 0) and out.kl[2] == 0 and out.kl[6] == 0


def _difference(f, x, d, h):
    return float(f(x + h * d) - f(x - h * d)) / (2 * h)


@pytest.mark.parametrize("what", ["policy", "preference", "distill"])
def test_gradient_against_differences(what):
    """Along a direction d: (L(x + h d) - L(x - h d)) / 2h. The loss comes back
    in fp32, off by 2^-24 of its size (below 4): 2^-22 / h = 2.4e-4 at h = 1e-3,
    and the third derivative's part, h^2 / 6 times a few, is below 1e-5."""
    g = _g(11)
    v = 12
    if what == "policy":
        x, y, old, adv, r = _policy_inputs(6, v, 8)
        lp = oracle.logp64(x, y[:, None], 1.0)[0][:, 0].float()
        old = lp + 0.05 * torch.sign(torch.randn(6, generator=g))  # ratios inside of the clip
        f = lambda z: lz.policy_loss(z, y, old, adv, ref_logp=r, kl_coef=0.3).loss  # noqa: E731
    elif what == "preference":
        x, y = torch.randn(4, 3, v, generator=g), torch.randint(0, v, (4, 3), generator=g)
        f = lambda z: lz.preference_loss(z, y, beta=0.5).loss  # noqa: E731
    else:
        x, ids = torch.randn(5, v, generator=g), torch.randint(0, v, (5, 4), generator=g)
        t = torch.randn(5, 4, generator=g)
        f = lambda z: lz.distill_loss(z, ids, t).loss  # noqa: E731
    x = x.requires_grad_(True)
    grad, = torch.autograd.grad(f(x), x)
    for seed in range(3):
        d = torch.randn(x.shape, generator=_g(seed))
        with torch.no_grad():
            got = _difference(f, x, d, 1e-3)
        assert abs(got - float((grad * d).sum())) < 1e-3


def test_rows_that_do_not_count_are_not_read():
    x, y, old, adv, r = _policy_inputs(6, 20, 1)
    x[2] = math.nan
    y[2] = -100
    x.requires_grad_(True)
    out = lz.policy_loss(x, y, old, adv, ref_logp=r, kl_coef=0.1)
    grad, = torch.autograd.grad(out.loss, x)
    assert torch.isfinite(out.loss) and torch.all(grad[2] == 0) and torch.isfinite(grad).all()
    w = torch.ones(6)
    w[2] = 0
    ids = torch.randint(0, 20, (6, 3), generator=_g(5))
    out = lz.distill_loss(x, ids, torch.zeros(6, 3), weights=w)
    grad, = torch.autograd.grad(out.loss, x)
    assert torch.isfinite(out.loss) and torch.all(grad[2] == 0) and torch.isfinite(grad).all()


def test_nothing_counts():
    x = torch.randn(3, 8, requires_grad=True)
    y = torch.full((3,), -100)
    z = torch.zeros(3)
    out = lz.policy_loss(x, y, z, z)
    assert out.loss == 0 and torch.all(torch.autograd.grad(out.loss, x)[0] == 0)
    out = lz.distill_loss(x, torch.full((3, 2), -1), torch.zeros(3, 2))
    assert out.loss == 0 and torch.all(torch.autograd.grad(out.loss, x)[0] == 0)
    assert torch.all(lz.token_logprobs(x, y) == 0)


def test_ids_beyond_the_vocabulary_show():
    x = torch.randn(3, 8)
    y = torch.tensor([1, 8, 2])
    assert lz.token_logprobs(x, y).isnan().tolist() == [False, True, False]
    z = torch.zeros(3)
    assert lz.policy_loss(x, y, z, z).loss.isnan()
    assert lz.distill_loss(x, y[:, None], z[:, None]).loss.isnan()


def test_denom():
    x, y, old, adv, _ = _policy_inputs(8, 20, 2, ref=False)
    a = lz.policy_loss(x, y, old, adv).loss * 8
    _close(lz.policy_loss(x, y, old, adv, denom=32).loss * 32, a, a.abs().double() + 8)
    _close(lz.policy_loss(x, y, old, adv, denom=torch.tensor(32)).loss * 32, a, a.abs().double() + 8)


X, Y, Z = torch.zeros(4, 10), torch.zeros(4, dtype=torch.long), torch.zeros(4)
T3, I3 = torch.zeros(4, 3), torch.zeros(4, 3, dtype=torch.long)
GRAD = torch.zeros(4, requires_grad=True)


@pytest.mark.parametrize("err,call", [
    (TypeError, lambda: lz.token_logprobs(X.double(), Y)),
    (TypeError, lambda: lz.token_logprobs(X.long(), Y)),
    (TypeError, lambda: lz.token_logprobs(X, Y.float())),
    (TypeError, lambda: lz.token_logprobs(X, Y.short())),
    (ValueError, lambda: lz.token_logprobs(X, Y[:3])),
    (ValueError, lambda: lz.token_logprobs(X, Y[:, None])),
    (ValueError, lambda: lz.token_logprobs(X[:, :0], Y)),
    (ValueError, lambda: lz.token_logprobs(torch.tensor(1.0), Y)),
    (ValueError, lambda: lz.token_logprobs(X, Y, temperature=0)),
    (ValueError, lambda: lz.token_logprobs(X, Y, temperature=-1.0)),
    (ValueError, lambda: lz.token_logprobs(X, Y, temperature=math.nan)),
    (ValueError, lambda: lz.token_logprobs(X, Y, temperature=math.inf)),
    (ValueError, lambda: lz.token_logprobs(X.to("meta"), Y.to("meta"))),
    (ValueError, lambda: lz.token_logprobs(X, Y.to("meta"))),
    (ValueError, lambda: lz.policy_loss(X, Y, Z[:3], Z)),
    (ValueError, lambda: lz.policy_loss(X, Y, Z, None)),
    (ValueError, lambda: lz.policy_loss(X, Y, GRAD, Z)),
    (ValueError, lambda: lz.policy_loss(X, Y, Z, Z, kl_coef=0.1)),
    (ValueError, lambda: lz.policy_loss(X, Y, Z, Z, clip_low=1.5)),
    (ValueError, lambda: lz.policy_loss(X, Y, Z, Z, clip_high=-0.1)),
    (ValueError, lambda: lz.policy_loss(X, Y, Z, Z, weights=Z[:2])),
    (ValueError, lambda: lz.policy_loss(X, Y, Z, Z, denom=0)),
    (ValueError, lambda: lz.policy_loss(X, Y, Z, Z, denom=torch.ones(2))),
    (TypeError, lambda: lz.policy_loss(X, Y, Y, Z)),
    (ValueError, lambda: lz.preference_loss(X, Y)),
    (ValueError, lambda: lz.preference_loss(X[None], Y[None])),
    (ValueError, lambda: lz.preference_loss(X.view(1, 4, 10).repeat(3, 1, 1), Y[None].repeat(3, 1))),
    (ValueError, lambda: lz.preference_loss(X, Y, cu_seqlens=torch.tensor([0, 4]))),
    (ValueError, lambda: lz.preference_loss(X, Y, cu_seqlens=torch.tensor([0, 2, 3, 4]))),
    (TypeError, lambda: lz.preference_loss(X, Y, cu_seqlens=torch.tensor([0., 2., 4.]))),
    (ValueError, lambda: lz.preference_loss(X, Y, cu_seqlens=torch.tensor([0, 2, 4]), ref_logp=Z)),
    (ValueError, lambda: lz.preference_loss(X, Y, cu_seqlens=torch.tensor([0, 2, 4]), label_smoothing=2)),
    (ValueError, lambda: lz.distill_loss(X, Y, Z)),
    (ValueError, lambda: lz.distill_loss(X, I3[:, :0], T3[:, :0])),
    (ValueError, lambda: lz.distill_loss(X, I3, T3[:, :2])),
    (ValueError, lambda: lz.distill_loss(X, torch.zeros(4, 1025, dtype=torch.long), torch.zeros(4, 1025))),
    (TypeError, lambda: lz.distill_loss(X, I3, T3.double())),
    (TypeError, lambda: lz.distill_loss(X, T3, T3)),
    (ValueError, lambda: lz.distill_loss(X, I3, T3.clone().requires_grad_(True))),
])
def test_refusals(err, call):
    with pytest.raises(err):
        call()


def test_offsets_that_do_not_rise_show():
    for off in ([0, 3, 2], [0, 2, 9], [-1, 2, 4]):
        assert lz.preference_loss(X, Y, cu_seqlens=torch.tensor(off)).loss.isnan()
