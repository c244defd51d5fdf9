"""Vocabulary losses on the GPU at the edges of what their arguments may hold:
ids beyond the vocabulary in rows that do not count, teachers without a finite
entry, scores far apart, saved tensors that come back in another layout, and
backward passes captured apart from their forward pass."""
import math

import pytest
import torch

import results_b200 as lz
from tests import _losses as oracle
from tests.test_losses_gpu import BF16, FP16, FP32, _check_distill, _check_policy, _distill_case, _gen, _logits, _policy_case, _tokens

pytestmark = pytest.mark.gpu

# rows that a part of a warp, a warp, a block and a cluster has, in the backward pass too
KERNELS = [(20000, 64, BF16), (6, 1000, BF16), (7, 30011, FP16), (6, 40000, BF16)]


@pytest.mark.parametrize("n,v,dtype", KERNELS)
def test_bad_tokens_of_rows_without_weight(n, v, dtype):
    """A padding id beyond the vocabulary in a row of weight zero: gradient zero, whatever the upstream."""
    x, y, old, adv, ref = _policy_case(n, v, dtype, 1)
    w = torch.ones(n, device="cuda")
    w[1] = w[n - 1] = 0
    bad = y.clone()
    bad[1], bad[n - 1] = v, 2**40
    x.requires_grad_(True)
    for up in (1.0, 2.0):
        up = torch.tensor(up, device="cuda")
        want, = torch.autograd.grad(lz.policy_loss(x, y, old, adv, ref_logp=ref, weights=w, kl_coef=0.1).loss, x, up)
        loss = lz.policy_loss(x, bad, old, adv, ref_logp=ref, weights=w, kl_coef=0.1).loss
        assert torch.isfinite(loss) and torch.isfinite(want).all()
        for _ in range(2):  # a second pass computes it anew
            grad, = torch.autograd.grad(loss, x, up, retain_graph=True)
            assert torch.equal(grad, want)
    # and one that counts is NaN in every way
    bad[0] = v
    loss = lz.policy_loss(x, bad, old, adv, weights=w).loss
    for up in (1.0, 2.0):
        grad, = torch.autograd.grad(loss, x, torch.tensor(up, device="cuda"), retain_graph=True)
        assert loss.isnan() and grad[0].isnan().all() and torch.isfinite(grad[1:]).all()


@pytest.mark.parametrize("n,v,dtype", KERNELS)
def test_bad_tokens_outside_of_the_sequences(n, v, dtype):
    """The tail of a packed buffer that nobody wrote, and log-probabilities that a user's loss leaves out."""
    x, y = _logits(n, v, dtype, 1).requires_grad_(True), _tokens(n, v, 2)
    cu = torch.tensor([1, 2, 3, 4, 5], device="cuda")
    bad = y.clone()
    bad[0], bad[5], bad[n - 1] = v, v + 5, 2**40
    for up in (1.0, 0.5):
        up = torch.tensor(up, device="cuda")
        want, = torch.autograd.grad(lz.preference_loss(x, y, cu_seqlens=cu).loss, x, up)
        loss = lz.preference_loss(x, bad, cu_seqlens=cu).loss
        grad, = torch.autograd.grad(loss, x, up)
        assert torch.isfinite(loss) and torch.equal(grad, want) and torch.all(grad[5:] == 0)
    logp = lz.token_logprobs(x, bad)
    grad, = torch.autograd.grad(torch.where(logp.isnan(), 0.0, logp).sum(), x)
    assert torch.all(grad[[0, 5, n - 1]] == 0) and torch.isfinite(grad).all() and logp.isnan().sum() == len({0, 5, n - 1})


@pytest.mark.parametrize("v", [40, 1003, 40000, 151552])
@pytest.mark.parametrize("k", [1, 5, 300])
@pytest.mark.parametrize("upstream", [1.0, 2.0])
def test_an_empty_list_shields_its_row(v, k, upstream):
    """A padding row is marked by its list alone; its logits are whatever was there."""
    x, ids, t = _distill_case(6, v, min(k, v), BF16, 3)
    x[1, v // 2], x[2, v // 3], x[3] = math.nan, math.inf, -math.inf
    ids[1:3] = -1
    t[3] = -math.inf
    leaf = x.clone().requires_grad_(True)
    out = lz.distill_loss(leaf, ids, t)
    grad, = torch.autograd.grad(out.loss, leaf, torch.tensor(upstream, device="cuda"))
    with torch.no_grad():
        assert torch.equal(lz.distill_loss(x, ids, t).kl[1:4], out.kl[1:4])
    assert torch.all(out.kl[1:4] == 0) and torch.all(grad[1:4] == 0)
    x[1:4] = 0  # the others are the formula's
    w = torch.tensor([1.0, 0, 0, 0, 1, 1], device="cuda")
    want = lz.distill_loss(x.requires_grad_(True), ids, t, weights=w, denom=6.0)
    assert torch.equal(want.loss, out.loss)
    assert torch.equal(grad, torch.autograd.grad(want.loss, x, torch.tensor(upstream, device="cuda"))[0])


@pytest.mark.parametrize("v", [40, 1003, 40000, 151552])
@pytest.mark.parametrize("k", [1, 5, 300])
@pytest.mark.parametrize("value", [math.nan, math.inf])
def test_a_teacher_without_a_number_shows(v, k, value):
    """One NaN or +inf among a row's entries, nothing else, and nothing else but padding or -inf; not in an
    entry that is padding, and not in a row without weight."""
    x, ids, t = _distill_case(7, v, min(k, v), FP32, 3)
    t[1, 0] = value
    t[2] = value
    t[3], ids[3, 1:] = value, -1
    t[4], t[4, 0] = -math.inf, value
    t[5, 0], ids[5, 0] = value, -1
    t[6] = value
    w = torch.ones(7, device="cuda")
    w[6] = 0
    leaf = x.requires_grad_(True)
    for upstream in (1.0, 2.0):
        out = lz.distill_loss(leaf, ids, t, weights=w)
        grad, = torch.autograd.grad(out.loss, leaf, torch.tensor(upstream, device="cuda"))
        assert out.loss.isnan() and out.kl.isnan().tolist() == [False, True, True, True, True, False, False]
        assert grad[1:5].isnan().all() and torch.isfinite(grad[[0, 5, 6]]).all()
    with torch.no_grad():
        assert torch.equal(lz.distill_loss(x, ids, t, weights=w).kl.isnan(), out.kl.isnan())


@pytest.mark.parametrize("v", [40, 40000])
@pytest.mark.parametrize("temperature", [0.25, 1.0, 3.0])
def test_a_teacher_at_its_types_ends(v, temperature):
    """Lists of the lowest value alone (all entries equal) or beside others, and of the largest."""
    x, ids, _ = _distill_case(4, v, 9, FP32, 3)
    for dtype in (FP32, BF16, FP16):
        low = torch.finfo(dtype).min
        t = torch.randn(4, 9, device="cuda", generator=_gen(1)).to(dtype)
        t[0] = low
        t[1, 3:] = low
        t[2] = -low
        t[3, 4], t[3, 5:] = -low, low
        _check_distill(x, ids, t, temperature=temperature)


@pytest.mark.parametrize("v", [40, 1003, 40000])
@pytest.mark.parametrize("low", [-100.0, -1000.0])
def test_a_watched_kl_changes_nothing(v, low):
    """kl_coef 0: the KL is an output alone, however far a token is below its reference."""
    x = _logits(4, v, FP32, 1)
    y = _tokens(4, v, 2)
    x[1, y[1]] = low
    x[2, y[2]] = -math.inf
    lp = oracle.logp64(x, y[:, None], 1.0)[0][:, 0]
    old, adv = torch.where(lp.isfinite(), lp, 0.0).float() + 0.1, torch.ones(4, device="cuda")
    x.requires_grad_(True)
    out = lz.policy_loss(x, y, old, adv, ref_logp=torch.full((4,), -1.0, device="cuda"))
    plain = lz.policy_loss(x, y, old, adv)
    assert torch.equal(out.loss, plain.loss) and torch.isfinite(out.loss) and out.kl[1] > 1e38 and out.kl[2] == math.inf
    for up in (1.0, 2.0):
        a, b = (torch.autograd.grad(o.loss, x, torch.tensor(up, device="cuda"), retain_graph=True)[0] for o in (out, plain))
        assert torch.isfinite(a).all() and torch.equal(a, b)


@pytest.mark.parametrize("v", [40, 1003, 40000])
def test_scores_far_apart(v):
    """Ratios and KL terms beyond fp32 that the advantage, the weight or the denominator brings back."""
    x, y, old, _, ref = _policy_case(6, v, FP32, 1)
    lp = oracle.logp64(x, y[:, None], 1.0)[0][:, 0]
    old, ref = (lp - 0.1).float(), (lp + 0.1).float()
    old[1], old[2], old[3], ref[4] = lp[1] - 100, lp[2] - 100, lp[3] + 200, lp[4] + 95
    adv = torch.tensor([1.0, 0.0, -1e-3, -1.0, 0.0, 2.0], device="cuda")
    z = x.requires_grad_(True)
    out = lz.policy_loss(z, y, old, adv, weights=torch.tensor([1.0, 1, 0, 1, 1, 1], device="cuda"))
    assert torch.isfinite(out.loss) and torch.isfinite(torch.autograd.grad(out.loss, z)[0]).all()
    want = oracle.policy(x.detach(), y, old, adv, ref, None, 0.2, 0.25, 0.5, 1.0, 1e35)["kl"]
    for upstream in (1.0, 2.0):
        out = lz.policy_loss(z, y, old, adv, ref_logp=ref, clip_low=0.2, clip_high=0.25, kl_coef=0.5, denom=1e35)
        grad, = torch.autograd.grad(out.loss, z, torch.tensor(upstream, device="cuda"))
        assert (out.kl == math.inf).tolist() == [False] * 4 + [True, False]  # as a number of 32 bits
        out = out._replace(kl=torch.where(out.kl.isinf(), want, out.kl.double()))
        _check_policy(x.detach(), y, old, adv, ref, beta=0.5, denom=1e35, upstream=upstream, out=out, grad=grad)


@pytest.mark.parametrize("v", [40, 40000])
@pytest.mark.parametrize("side", [0, 1])
def test_preference_with_an_impossible_token(v, side):
    """A token of probability zero in one answer: the margin is infinite. Without smoothing the loss has one
    term, which is zero (a rejected answer that cannot be) or infinite."""
    x = _logits(4, v, FP32, 1)
    y = _tokens(4, v, 2)
    x[2 * side, y[2 * side]] = -math.inf
    x.requires_grad_(True)
    for eps in (0.0, 1.0):
        out = lz.preference_loss(x.view(2, 2, v), y.view(2, 2), label_smoothing=eps)
        zero = side == (1 if eps == 0.0 else 0)
        assert float(out.loss.detach()) == (0.0 if zero else math.inf)
        grad, = torch.autograd.grad(out.loss, x)
        assert torch.isfinite(grad).all() and bool((grad == 0).all()) == zero


@pytest.mark.parametrize("v", [301, 40000])
def test_saved_logits_may_come_back_in_another_layout(v):
    """Offloaded logits that come back contiguous, to the address that their strided view had."""
    y = _tokens(12, v, 2).view(3, 4)
    old, adv = torch.randn(2, 3, 4, device="cuda", generator=_gen(3)) - 5
    ids = torch.randint(0, v, (3, 4, 5), device="cuda", generator=_gen(4))
    t = torch.randn(3, 4, 5, device="cuda", generator=_gen(5))
    store = _logits(15, v, BF16, 1).view(3, 5, v)

    def step(hooked):
        base = store.clone().requires_grad_(True)
        z = base * 1  # not a leaf: only the view below is kept
        view = z[:, :-1]
        if not hooked:
            return base, view, None

        def pack(s):
            return s.contiguous().clone(), s.data_ptr() == view.data_ptr() and s.dim() == 3

        def unpack(p):
            if not p[1]:
                return p[0].clone()
            flat = z.detach().view(-1)[:p[0].numel()].view(p[0].shape)
            assert flat.data_ptr() == view.data_ptr()
            return flat.copy_(p[0])

        return base, view, torch.autograd.graph.saved_tensors_hooks(pack, unpack)

    for f in (lambda x: lz.policy_loss(x, y, old, adv).loss, lambda x: lz.distill_loss(x, ids, t).loss,
              lambda x: lz.token_logprobs(x, y).sum(),
              lambda x: lz.preference_loss(x[:2], y[:2]).loss):
        grads = []
        for hooked in (False, True):
            base, view, hooks = step(hooked)
            if hooks:
                with hooks:
                    loss = f(view) * 3
            else:
                loss = f(view) * 3
            grads += torch.autograd.grad(loss, base)
        assert torch.equal(*grads)


def test_saved_tensors_may_come_back_with_other_strides():
    """Tokens and lists that are not contiguous any more; a tensor that stays on the host is refused."""
    x, ids, t = _distill_case(6, 1003, 5, BF16, 3)
    y = ids[:, 0].contiguous()
    x.requires_grad_(True)

    def spread(s):
        wide = torch.zeros(*s.shape, 2, dtype=s.dtype, device=s.device)
        wide[..., 0] = s.detach()
        return wide[..., 0]

    def shift(s):  # behind one element of a buffer
        return torch.cat([s.detach().reshape(-1)[:1], s.detach().reshape(-1)])[1:].view(s.shape)

    for f in (lambda: lz.token_logprobs(x, y).sum(), lambda: lz.distill_loss(x, ids, t).loss):
        want, = torch.autograd.grad(f() * 2, x)
        for pack in (spread, shift):
            with torch.autograd.graph.saved_tensors_hooks(pack, lambda s: s):
                loss = f() * 2
            assert torch.equal(torch.autograd.grad(loss, x)[0], want)
        with torch.autograd.graph.saved_tensors_hooks(lambda s: s.cpu(), lambda s: s):
            loss = f() * 2
        with pytest.raises(RuntimeError, match="saved"):
            torch.autograd.grad(loss, x)


@pytest.mark.parametrize("v", [700, 40000])
@pytest.mark.parametrize("kind", ["policy", "distill"])
def test_backward_captured_apart(v, kind):
    """A backward pass in a graph of its own gives the formula's gradient at every replay, whatever was done to
    the last one and whatever upstream that had; its forward pass ran eagerly or in another graph."""
    x, y, old, adv, ref = _policy_case(12, v, BF16, 2)
    x, ids, t = _distill_case(12, v, 9, BF16, 2)
    x.requires_grad_(True)

    def f():
        if kind == "policy":
            return lz.policy_loss(x, y, old, adv, ref_logp=ref, kl_coef=0.1).loss
        return lz.distill_loss(x, ids, t).loss

    want = {u: torch.autograd.grad(f(), x, torch.tensor(u, device="cuda"))[0] for u in (1.0, 2.0)}
    for captured in (False, True):
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):  # a pass before the capture, as every graph has it
            torch.autograd.grad(f(), x)
            if not captured:
                loss = f()
        torch.cuda.current_stream().wait_stream(side)
        if captured:
            first = torch.cuda.CUDAGraph()
            with torch.cuda.graph(first, stream=side):
                loss = f()
            first.replay()
        up = torch.ones((), device="cuda")
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            grad, = torch.autograd.grad(loss, x, up, retain_graph=True)
            half = grad * 0.5
            grad.mul_(4)
        for u in (1.0, 2.0, 1.0, 1.0):
            up.fill_(u)
            graph.replay()
            assert torch.equal(grad, want[u] * 4) and torch.equal(half, want[u] * 0.5)
    # and a captured forward pass with an eager backward pass: a replay writes over no gradient that was given out
    first.replay()
    first.replay()
    g2 = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g2):
        loss2 = f()
    g2.replay()
    a, = torch.autograd.grad(loss2, x, retain_graph=True)
    a.zero_()
    g2.replay()
    assert torch.all(a == 0)
    assert torch.equal(torch.autograd.grad(loss2, x)[0], want[1.0])


def test_forward_mode_and_tracing_are_refused():
    """Neither a tangent nor a recorded graph is lost without a word."""
    from torch.autograd import forward_ad

    x, ids, t = _distill_case(4, 300, 5, FP32, 3)
    y = ids[:, 0].contiguous()
    z = torch.zeros(4, device="cuda")
    calls = [lambda x, z: lz.token_logprobs(x, y), lambda x, z: lz.policy_loss(x, y, z, z + 1).loss,
             lambda x, z: lz.preference_loss(x.view(2, 2, 300), y.view(2, 2)).loss,
             lambda x, z: lz.distill_loss(x, ids, t, weights=z + 1).loss]
    for f in calls:
        for needs_grad in (False, True):
            leaf = x.clone().requires_grad_(needs_grad)
            with forward_ad.dual_level():
                with pytest.raises(RuntimeError, match="forward-mode"):
                    f(forward_ad.make_dual(leaf, torch.ones_like(x)), z)
                assert torch.equal(f(leaf, z), f(leaf, z))  # nothing to lose: as ever
            with pytest.raises(RuntimeError, match="traced"):
                torch.jit.trace(lambda a: f(a, z), (leaf,), check_trace=False)
    with forward_ad.dual_level(), pytest.raises(RuntimeError, match="forward-mode"):
        calls[1](x, forward_ad.make_dual(z, torch.ones_like(z)))


@pytest.mark.parametrize("wait_ns", [1, 2])
@pytest.mark.parametrize("n,v,dtype", [(6, 151552, BF16), (40, 151936, FP32), (700, 70001, FP16)])
def test_waits_that_give_up(monkeypatch, wait_ns, n, v, dtype):
    """With next to no time to wait for a copy or a peer: whatever is not the very value of an ordinary call is
    NaN, a row's log-probability together with all of its gradient, and the next call is an ordinary one again."""
    from results_b200.ops import losses

    x, y, old, adv, ref = _policy_case(n, v, dtype, 1)
    y[n // 2] = -1
    ids, t = torch.randint(0, v, (n, 70), device="cuda", generator=_gen(1)), torch.randn(n, 70, device="cuda", generator=_gen(2))
    x.requires_grad_(True)

    def step():
        a, d = lz.policy_loss(x, y, old, adv, ref_logp=ref, kl_coef=0.1), lz.distill_loss(x, ids, t)
        b, lp = lz.preference_loss(x.view(2, n // 2, v), y.view(2, -1)), lz.token_logprobs(x, y)
        res = {"policy": (a.loss, a.logp), "distill": (d.loss, d.kl), "preference": (b.loss, None), "logp": (lp.sum(), lp)}
        return {k: (*r, *(torch.autograd.grad(r[0], x, torch.tensor(u, device="cuda"), retain_graph=u == 1)[0] for u in (1.0, 2.0)))
                for k, r in res.items()}

    want = step()
    launch = losses._launch

    def short(fn, args):
        if fn != "lz_loss_pairs":
            args.wait_ns = wait_ns
        return launch(fn, args)

    monkeypatch.setattr(losses, "_launch", short)
    got = step()
    monkeypatch.setattr(losses, "_launch", launch)
    again = step()
    torch.cuda.synchronize()
    for k in want:
        for a, b, c in zip(want[k], got[k], again[k]):
            assert a is None or (torch.equal(a, c) and bool(((a == b) | b.isnan()).all())), k
        loss, rows, fused, other = got[k]
        if rows is not None:
            lost = rows.isnan()
            print(k, n, v, wait_ns, "rows that were lost:", int(lost.sum()), "loss", float(loss.detach()))
            counted = y >= 0 if k != "distill" else y == y
            assert not (loss.isnan() and not lost.any())
            if k in ("policy", "distill"):
                assert torch.equal(fused.isnan().all(1), fused.isnan().any(1)) and fused[lost].isnan().all()
            assert other[lost & counted].isnan().all()


@pytest.mark.parametrize("n,v,dtype", [(40, 151552, BF16), (7, 151936, FP32), (3000, 24000, BF16), (20000, 64, BF16)])
def test_losses_inside_an_sm_budget(n, v, dtype):
    """On the stream of a few SMs, where the clusters take turns: the same bits."""
    from results_b200.utils.sm_budget import SmBudget

    x, y, old, adv, ref = _policy_case(n, v, dtype, 1)
    y[n // 2] = -1
    ids, t = torch.randint(0, v, (n, 20), device="cuda", generator=_gen(1)), torch.randn(n, 20, device="cuda", generator=_gen(2))
    x.requires_grad_(True)

    def step():
        losses = [lz.policy_loss(x, y, old, adv, ref_logp=ref, kl_coef=0.1).loss, lz.distill_loss(x, ids, t).loss,
                  lz.token_logprobs(x, y).sum()]
        return losses + [torch.autograd.grad(loss * s, x)[0] for loss, s in zip(losses, (1, 2, 3))]

    want = step()
    torch.cuda.synchronize()
    with SmBudget(0, 16) as b:
        with torch.cuda.stream(b.stream):
            got = step()
        b.stream.synchronize()
        assert all(torch.equal(a, c) for a, c in zip(want, got))
        del got


@pytest.mark.parametrize("v", [40, 40000])
def test_a_small_kl_beside_a_far_ratio(v):
    """A ratio beyond fp32 at advantage zero, and a reference that is close: the gradient is the KL's."""
    x, y, _, _, _ = _policy_case(3, v, FP32, 1)
    lp = oracle.logp64(x, y[:, None], 1.0)[0][:, 0]
    ref = (lp + torch.tensor([1e-4, 1e-2, -1.0], device="cuda")).float()
    old, adv = (lp - 120).float(), torch.zeros(3, device="cuda")
    _check_policy(x, y, old, adv, ref, beta=0.5)
    _check_policy(x, y, old, adv, ref, beta=0.5, upstream=-3.0)


def test_calls_inside_a_compiled_function():
    """The compiler runs them as they are (its eager backend: nothing else of the function matters here)."""
    w, h = torch.randn(64, 1000, device="cuda", generator=_gen(1)), torch.randn(8, 64, device="cuda", generator=_gen(2))
    w.requires_grad_(True)
    y, z = torch.arange(8, device="cuda"), torch.zeros(8, device="cuda")
    ids, t = y[:, None] + torch.arange(5, device="cuda"), torch.randn(8, 5, device="cuda", generator=_gen(3))
    for f in (lambda w: lz.policy_loss(h @ w, y, z - 7, z + 1, ref_logp=z - 7, kl_coef=0.1).loss * 2,
              lambda w: -lz.token_logprobs(h @ w, y).mean(), lambda w: lz.distill_loss(h @ w, ids, t).loss,
              lambda w: lz.preference_loss((h @ w).view(2, 4, 1000), y.view(2, 4)).loss):
        c = torch.compile(f, backend="eager")
        assert torch.equal(c(w), f(w))
        assert torch.equal(torch.autograd.grad(c(w), w)[0], torch.autograd.grad(f(w), w)[0])
        with torch.no_grad():
            assert torch.equal(c(w), f(w))
