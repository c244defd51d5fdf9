"""Vocabulary losses on CPU tensors at the edges of what their arguments may hold."""
import math

import pytest
import torch

import results_b200 as lz


def _g(seed):
    return torch.Generator().manual_seed(seed)


def _inputs(n, v, seed=1):
    x = torch.randn(n, v, generator=_g(seed)).requires_grad_(True)
    return x, torch.randint(0, v, (n,), generator=_g(seed + 1)), torch.zeros(n)


def test_gradients_of_ids_beyond_the_vocabulary():
    """NaN in the rows that count, zero in those that do not."""
    x, y, z = _inputs(6, 8)
    y[1], y[2] = 8, 2**40
    w = torch.tensor([1.0, 1, 0, 1, 1, 1])
    for up in (1.0, 2.0):
        out = lz.token_logprobs(x, y)
        grad, = torch.autograd.grad((out * up).sum(), x)
        assert grad[1:3].isnan().all() and torch.isfinite(grad[[0, 3, 4, 5]]).all()
        out = lz.policy_loss(x, y, z, z + 1, weights=w)
        grad, = torch.autograd.grad(out.loss * up, x)
        assert out.loss.isnan() and grad[1].isnan().all() and torch.isfinite(grad[[0, 3, 4, 5]]).all() and torch.all(grad[2] == 0)
        out = lz.preference_loss(x, y, cu_seqlens=torch.tensor([3, 4, 6]))
        grad, = torch.autograd.grad(out.loss * up, x)
        assert torch.isfinite(out.loss) and torch.isfinite(grad).all() and torch.all(grad[:3] == 0)
        ids = torch.stack([torch.zeros_like(y), y], 1)
        t = torch.zeros(6, 2)
        t[1, 1] = -math.inf  # an entry of no weight is looked at all the same
        out = lz.distill_loss(x, ids, t, weights=w)
        grad, = torch.autograd.grad(out.loss * up, x)
        assert out.kl.isnan().tolist() == [False, True, False, False, False, False]
        assert grad[1].isnan().all() and torch.isfinite(grad[[0, 3, 4, 5]]).all() and torch.all(grad[2] == 0)
    logp = lz.token_logprobs(x, y)
    grad, = torch.autograd.grad(torch.where(logp.isnan(), 0.0, logp).sum(), x)
    assert torch.all(grad[1:3] == 0) and torch.isfinite(grad).all()


def test_gradient_of_a_teacher_without_a_number():
    x, y, _ = _inputs(5, 8)
    ids = torch.stack([y, (y + 1) % 8, (y + 2) % 8], 1)
    for value in (math.nan, math.inf):
        t = torch.randn(5, 3, generator=_g(3))
        t[1, 0] = value
        t[2] = value
        t[3, 1], ids[3, 1] = value, -1  # padding
        t[4] = value
        out = lz.distill_loss(x, ids, t, weights=torch.tensor([1.0, 1, 1, 1, 0]))
        grad, = torch.autograd.grad(out.loss, x)
        assert out.kl.isnan().tolist() == [False, True, True, False, False]
        assert grad[1:3].isnan().all() and torch.isfinite(grad[[0, 3, 4]]).all() and torch.all(grad[4] == 0)


def test_an_empty_list_shields_its_row():
    x, y, _ = _inputs(5, 8)
    with torch.no_grad():
        x[1, 3], x[2, 4], x[3] = math.nan, math.inf, -math.inf
    ids, t = torch.stack([y, (y + 1) % 8], 1), torch.randn(5, 2, generator=_g(3))
    ids[1:3], t[3] = -1, -math.inf
    out = lz.distill_loss(x, ids, t)
    grad, = torch.autograd.grad(out.loss, x)
    assert torch.isfinite(out.loss) and torch.all(out.kl[1:4] == 0) and torch.all(grad[1:4] == 0) and torch.isfinite(grad).all()


def test_a_watched_kl_changes_nothing():
    x, y, z = _inputs(4, 8)
    with torch.no_grad():
        x[1, y[1]], x[2, y[2]] = -1000, -math.inf
    out = lz.policy_loss(x, y, z - 2, z + 1, ref_logp=z - 1)
    plain = lz.policy_loss(x, y, z - 2, z + 1)
    assert torch.equal(out.loss, plain.loss) and torch.isfinite(out.loss) and torch.all(out.kl[1:3] == math.inf)
    a, b = (torch.autograd.grad(o.loss, x)[0] for o in (out, plain))
    assert torch.isfinite(a).all() and torch.equal(a, b)


@pytest.mark.parametrize("side", [0, 1])
def test_preference_with_an_impossible_token(side):
    x, y, _ = _inputs(4, 8)
    with torch.no_grad():
        x[2 * side, y[2 * side]] = -math.inf
    for eps in (0.0, 1.0):
        out = lz.preference_loss(x.view(2, 2, 8), y.view(2, 2), label_smoothing=eps)
        zero = side == (1 if eps == 0.0 else 0)
        assert float(out.loss.detach()) == (0.0 if zero else math.inf)
        grad, = torch.autograd.grad(out.loss, x)
        assert torch.isfinite(grad).all() and bool((grad == 0).all()) == zero


def test_a_default_device_of_another_kind():
    """Tensors go by the logits' device, whatever torch's default is."""
    x, y, z = _inputs(6, 8)
    y[1] = 8
    w = torch.tensor([1.0, 0, 1, 1, 1, 1])
    cu, ids, t = torch.tensor([0, 3, 2, 4, 5]), y.clamp(max=7)[:, None], torch.zeros(6, 1)

    def run():
        outs = [lz.token_logprobs(x, y), lz.policy_loss(x, y, z, z + 1, ref_logp=z, weights=w, denom=4.0).loss,
                lz.distill_loss(x, ids, t).loss, lz.preference_loss(x, y, cu_seqlens=cu).loss]
        return [o.detach() for o in outs] + [torch.autograd.grad(o.nan_to_num().sum(), x)[0] for o in outs]

    want = run()
    torch.set_default_device("meta")
    try:
        got = run()
    finally:
        torch.set_default_device(None)
    for a, b in zip(want, got):
        assert torch.equal(a.nan_to_num(), b.nan_to_num())
