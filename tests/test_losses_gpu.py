"""Vocabulary losses on the GPU against their formulas in 64 bits: types, sizes
that split in every way, strides, masked values, empty rows, upstream gradients,
captured graphs, other streams, and a run of them together. The bounds come
from the number of roundings (tests/_losses.py)."""
import math

import pytest
import torch

import results_b200 as lz
from tests import _losses as oracle

pytestmark = pytest.mark.gpu

BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32
# rows, vocabulary, type: one row and many, vocabularies below, at and beside the vectors' and the
# blocks' sizes, odd ones, the largest of the models the package knows
SIZES = [(1, 1, FP32), (3, 2, BF16), (5, 7, FP16), (2, 8, BF16), (700, 9, BF16), (4, 255, FP32), (33, 1000, BF16),
         (6, 4096, FP16), (5, 4097, BF16), (3, 12289, FP32), (149, 32003, FP16), (7, 50021, BF16), (2, 50021, FP32),
         (1, 151552, BF16), (160, 151552, BF16), (2, 151936, FP32), (75, 151936, FP32), (1, 262144, BF16),
         (2, 1000003, BF16), (1, 600011, FP32)]


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _logits(n, v, dtype, seed, std=2.5):
    return torch.randn(n, v, device="cuda", generator=_gen(seed), dtype=dtype) * std


def _tokens(n, v, seed, x=None):
    if x is not None and n * v < 4_000_000:  # likely tokens
        u = torch.rand(n, v, device="cuda", generator=_gen(seed))
        return (x.float() - u.log().neg().log()).argmax(1)
    return torch.randint(0, v, (n,), device="cuda", generator=_gen(seed))


def _near(got, want, off, what):
    d = (got.double() - want).abs()
    # a bound that is not finite says that the value is not finite either
    bad = ~((d <= off) | (got.double() == want) | (got.isnan() & want.isnan()))
    assert not bad.any(), (what, int(bad.sum()), float((d / off)[bad].max()))


def _policy_case(n, v, dtype, seed, ref=True, temperature=1.0, x=None):
    x = _logits(n, v, dtype, seed) if x is None else x
    y = _tokens(n, v, seed + 1, x)
    lp = oracle.logp64(x, y[:, None], temperature)[0][:, 0]
    d = torch.randn(n, device="cuda", generator=_gen(seed + 2), dtype=torch.float64) * 0.2
    for edge in (math.log(0.8), math.log(1.25)):  # at the border itself the gradient is one or the other
        d = torch.where((d - edge).abs() < 1e-3, d + 4e-3, d)
    adv = torch.randn(n, device="cuda", generator=_gen(seed + 3))
    r = (lp + 0.3 * torch.randn(n, device="cuda", generator=_gen(seed + 4))).float() if ref else None
    return x, y, (lp - d).float(), adv, r


def _check_policy(x, y, old, adv, ref, w=None, beta=0.1, temperature=1.0, denom=None, upstream=1.0, out=None, grad=None):
    leaf = x.detach().requires_grad_(True) if out is None else None
    if out is None:
        out = lz.policy_loss(leaf, y, old, adv, ref_logp=ref, weights=w, clip_low=0.2, clip_high=0.25,
                             kl_coef=beta if ref is not None else 0.0, temperature=temperature, denom=denom)
        grad, = torch.autograd.grad(out.loss, leaf, torch.tensor(upstream, device="cuda"))
    want = oracle.policy(x.detach(), y, old, adv, ref, w, 0.2, 0.25, beta if ref is not None else 0.0, temperature, denom)
    off = oracle.logp_off(x, temperature, want["logp"])
    _near(out.logp, want["logp"], off, "logp")
    assert torch.equal(out.clipped, want["clipped"])
    each_off = want["bend"].abs() * temperature * off + 2.0 ** -22 * (want["each"] * want["scale"]).abs()
    if ref is not None:
        d = ref.double() - want["logp"]
        kl_off = d.expm1().abs() * off + off * off + 2.0 ** -24 * want["kl"]
        _near(out.kl, want["kl"], kl_off, "kl")
        each_off = each_off + (want["scale"] * beta * kl_off).abs()
    _near(out.loss, want["loss"], each_off.sum() + 2.0 ** -22 * want["loss"].abs() + 1e-30, "loss")
    want["grad"], want["slope"] = want["grad"] * upstream, want["slope"] * upstream
    _near(grad, want["grad"], oracle.grad_off(want, x.dtype, off, (want["bend"] * upstream).abs() * off), "grad")
    return out, grad


@pytest.mark.parametrize("n,v,dtype", SIZES)
def test_policy_sizes(n, v, dtype):
    _check_policy(*_policy_case(n, v, dtype, n + v))


@pytest.mark.parametrize("n,v,dtype", SIZES)
def test_token_logprobs_sizes(n, v, dtype):
    x = _logits(n, v, dtype, n * v).requires_grad_(True)
    y = _tokens(n, v, 5, x.detach())
    y[n // 3] = -1
    out = lz.token_logprobs(x, y)
    on = (y >= 0).double()
    lp, p = oracle.logp64(x.detach(), y.clamp(min=0)[:, None], 1.0)
    off = oracle.logp_off(x.detach(), 1.0, lp[:, 0])
    _near(out, lp[:, 0] * on, off, "logp")
    with torch.no_grad():
        assert torch.equal(lz.token_logprobs(x, y), out)
    up = torch.randn(n, device="cuda", generator=_gen(3))
    grad, = torch.autograd.grad(out, x, up)
    want = -p
    want[torch.arange(n, device="cuda"), y.clamp(min=0)] += 1
    slope = up.double() * on
    _near(grad, want * slope[:, None], oracle.grad_off({"p": p, "slope": slope, "grad": want * slope[:, None]}, dtype,
                                                       off, torch.zeros_like(off)), "grad")


def _distill_case(n, v, k, dtype, seed):
    k = min(k, v)
    x = _logits(n, v, dtype, seed)
    ids = torch.stack([torch.randperm(v, device="cuda", generator=_gen(seed + r))[:k] for r in range(min(n, 16))])
    ids = ids[torch.arange(n, device="cuda") % len(ids)]
    t = (torch.randn(n, k, device="cuda", generator=_gen(seed + 1)) * 3).to(dtype)
    return x, ids, t


def _check_distill(x, ids, t, w=None, temperature=1.0, denom=None, upstream=1.0):
    leaf = x.detach().requires_grad_(True)
    out = lz.distill_loss(leaf, ids, t, weights=w, temperature=temperature, denom=denom)
    grad, = torch.autograd.grad(out.loss, leaf, torch.tensor(upstream, device="cuda"))
    want = oracle.distill(x, ids, t, w, temperature, denom)
    some = want["slope"] != 0
    k = ids.shape[1]
    # q: its exponential (2 steps), exponent (half a step of at most 2 max |t|) and sum (k half steps at
    # most); an entry at -inf has no error, its q is zero, so |t| is that of the others
    tz = torch.where((ids >= 0) & t.isfinite(), t.double().abs() / temperature, 0.0).amax(1)
    q_off = 2.0 ** -24 * (k / 16 + 16 + 4 * tz)
    lp = oracle.logp64(x, ids.clamp(min=0), temperature)[0]
    span = torch.where(lp.isfinite(), lp.abs(), 0.0).amax(1) + tz * 2 + math.log(k)
    off = oracle.logp_off(x, temperature, lp.abs().amax(1).clamp(max=1e30))
    kl_off = torch.where(some, off + q_off * (span + 2), 0.0) + 2.0 ** -24 * want["kl"]
    _near(out.kl, want["kl"], kl_off, "kl")
    _near(out.loss, want["loss"], (kl_off * want["scale"].abs()).sum() + 2.0 ** -22 * want["loss"].abs() + 1e-30, "loss")
    want["grad"], want["slope"] = want["grad"] * upstream, want["slope"] * upstream
    q = torch.where(want["slope"][:, None] != 0, want["p"] - want["grad"] / -want["slope"][:, None], 0.0)
    bound = oracle.grad_off(want, x.dtype, off, torch.zeros_like(off))
    _near(grad, want["grad"], bound + (want["slope"].abs() * q_off)[:, None] * q.abs() * 1.01, "grad")
    return out, grad


@pytest.mark.parametrize("n,v,dtype", SIZES)
@pytest.mark.parametrize("k", [1, 20, 300])
def test_distill_sizes(n, v, dtype, k):
    _check_distill(*_distill_case(n, v, k, dtype, n + v + k))


def _check_preference(x, y, ref, ends, shape=None, cu=None, eps=0.1, normalized=False, upstream=1.0, temperature=1.0):
    leaf = x.detach().requires_grad_(True)
    a, b = (leaf, y) if shape is None else (leaf.view(*shape, -1), y.view(shape))
    out = lz.preference_loss(a, b, ref_logp=ref, cu_seqlens=cu, label_smoothing=eps, length_normalized=normalized,
                             temperature=temperature)
    grad, = torch.autograd.grad(out.loss, leaf, torch.tensor(upstream, device="cuda"))
    want = oracle.preference(x, y, ref, ends, 0.1, eps, normalized, temperature)
    off = torch.where(y >= 0, oracle.logp_off(x, temperature, want["logp"]), 0.0)
    per = [1.0 / max(1, int((y[i:j] >= 0).sum())) if normalized else 1.0 for i, j in zip(ends, ends[1:])]
    r_off = 0.1 * torch.stack([off[i:j].sum() * f for (i, j), f in zip(zip(ends, ends[1:]), per)])
    r_off = r_off + 2.0 ** -24 * want["rewards"].abs()
    k = len(want["h"])
    _near(out.chosen_rewards, want["rewards"][:k], r_off[:k], "chosen")
    _near(out.rejected_rewards, want["rewards"][k:], r_off[k:], "rejected")
    h_off = r_off[:k] + r_off[k:]
    _near(out.loss, want["loss"], h_off.mean() + 2.0 ** -24 * want["loss"], "loss")
    # the slope's derivative in h is at most beta / (4 pairs); it is rounded to fp32
    slope_off = torch.zeros(len(y), device="cuda", dtype=torch.float64)
    for i, (s, e) in enumerate(zip(ends, ends[1:])):
        slope_off[s:e] = 0.1 / k / 4 * h_off[i % k] * per[i] / temperature
    slope_off = slope_off * abs(upstream) + 2.0 ** -23 * want["slope"].abs() * abs(upstream)
    want["grad"], want["slope"] = want["grad"] * upstream, want["slope"] * upstream
    _near(grad, want["grad"], oracle.grad_off(want, x.dtype, off, slope_off), "grad")


@pytest.mark.parametrize("v,dtype", [(50, FP32), (1001, FP16), (32003, BF16), (151936, BF16)])
@pytest.mark.parametrize("normalized", [False, True])
@pytest.mark.parametrize("ids", [torch.int64, torch.int32])
def test_preference(v, dtype, normalized, ids):
    pairs, length = 3, 7
    n = 2 * pairs * length
    x = _logits(n, v, dtype, v)
    y = _tokens(n, v, 4).to(ids)
    y[torch.rand(n, device="cuda", generator=_gen(8)) < 0.3] = -100
    y[:length] = -100  # a sequence with no token that counts
    ref = torch.randn(2 * pairs, device="cuda", generator=_gen(9)) * 3
    _check_preference(x, y, ref, [i * length for i in range(2 * pairs + 1)], shape=(2 * pairs, length), normalized=normalized)
    ends = [2, 9, 9, 10, 30, 31, 40]
    _check_preference(x, y, None, ends, cu=torch.tensor(ends, device="cuda", dtype=ids), normalized=normalized,
                      upstream=0.25, temperature=0.7, eps=0.0)


def test_preference_long_sequences_and_many_pairs():
    x = _logits(6000, 64, BF16, 1)
    y = _tokens(6000, 64, 2)
    _check_preference(x, y, None, [0, 2999, 6000], cu=torch.tensor([0, 2999, 6000], device="cuda"))
    ends = list(range(0, 6001, 3))
    _check_preference(x, y, None, ends, shape=(2000, 3))


def test_preference_offsets_that_do_not_rise():
    x, y = _logits(8, 40, FP32, 1).requires_grad_(True), _tokens(8, 40, 2)
    for off in ([0, 5, 4], [0, 4, 9], [-3, 4, 8], [0, 2**31 - 1, 2**31 - 1]):
        out = lz.preference_loss(x, y, cu_seqlens=torch.tensor(off, device="cuda"))
        assert out.loss.isnan()
        torch.autograd.grad(out.loss, x)


# ---- layouts --------------------------------------------------------------------------------------------


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("v", [96, 1003, 40961])
@pytest.mark.parametrize("layout", ["shifted", "columns", "offset", "transposed", "four", "expanded", "one"])
def test_layouts(dtype, v, layout):
    """Every layout gives the formula's values."""
    base = _logits(24, v, dtype, 7)
    if layout == "shifted":  # [batch, length, vocab] without each sequence's last position
        store = torch.zeros(4, 7, v, device="cuda", dtype=dtype)
        store[:, :-1] = base.view(4, 6, v)
        x, shape = store[:, :-1], (4, 6)
    elif layout == "columns":  # part of a wider head
        store = torch.full((24, v + 37), 30.0, device="cuda", dtype=dtype)
        store[:, 5:5 + v] = base
        x, shape = store[:, 5:5 + v], (24,)
    elif layout == "offset":  # a flat buffer from an odd element on
        store = torch.empty(24 * v + 3, device="cuda", dtype=dtype)
        x, shape = store[3:].view(24, v).copy_(base), (24,)
    elif layout == "transposed":  # a vocabulary that is not contiguous
        x, shape = base.t().contiguous().t(), (24,)
    elif layout == "four":
        x, shape = base.view(2, 3, 4, v).transpose(0, 1).contiguous().transpose(0, 1), (2, 3, 4)
    elif layout == "expanded":
        base = base[:1].expand(24, v)
        x, shape = base.view(4, 6, v), (4, 6)
    else:
        base = base[:1]
        x, shape = base[0], ()
    n = math.prod(shape)
    y, old, adv, r = _policy_case(n, v, dtype, 7, x=base.contiguous())[1:]
    leaf = x.detach().requires_grad_(True)
    out = lz.policy_loss(leaf, y.view(shape), old.view(shape), adv.view(shape), ref_logp=r.view(shape), clip_low=0.2,
                         clip_high=0.25, kl_coef=0.1)
    grad, = torch.autograd.grad(out.loss, leaf)
    assert grad.shape == x.shape and out.logp.shape == tuple(shape)
    flat = type(out)(out.loss, *(t.view(-1) for t in out[1:]))
    _check_policy(base.contiguous(), y, old, adv, r, out=flat, grad=grad.reshape(n, v))
    up = torch.randn(shape, device="cuda", generator=_gen(1))
    lp = lz.token_logprobs(leaf, y.view(shape).int())
    # each is within the bound of the formula, so they are within twice that of each other (a row
    # that has a gradient to give may be added up in another order than one that has none)
    off = oracle.logp_off(base.contiguous(), 1.0, out.logp.view(-1).double())
    _near(lp.view(-1), out.logp.view(-1).double(), 2 * off, "logp")
    g2, = torch.autograd.grad(lp, leaf, up)
    assert torch.equal(g2.reshape(n, v), _plain_grad(base.contiguous(), y, up.view(-1), g2.reshape(n, v)))


def _plain_grad(x, y, up, got):
    """`got`, if it is within the bound of the formula; what the formula gives otherwise."""
    lp, p = oracle.logp64(x, y[:, None], 1.0)
    want = -p
    want[torch.arange(len(y), device="cuda"), y] += 1
    want = want * up.double()[:, None]
    off = oracle.grad_off({"p": p, "slope": up.double(), "grad": want}, x.dtype, oracle.logp_off(x, 1.0, lp[:, 0]),
                          torch.zeros_like(lp[:, 0]))
    return got if bool(((got.double() - want).abs() <= off).all()) else want


def test_rows_apart_by_more_than_32_bits():
    """Two rows of one storage, 2^31 elements and more apart."""
    v = 1 << 20
    store = torch.zeros(2100, v, device="cuda", dtype=torch.float16)  # 4.4 GB
    store[0] = _logits(1, v, FP16, 1)[0]
    store[2099] = _logits(1, v, FP16, 2)[0]
    x = store[::2099]
    y = _tokens(2, v, 3)
    out = lz.token_logprobs(x, y)
    lp, _ = oracle.logp64(x, y[:, None], 1.0)
    _near(out, lp[:, 0], oracle.logp_off(x, 1.0, lp[:, 0]), "logp")
    # and a gradient that is larger than that
    leaf = store.requires_grad_(True)
    z = torch.zeros(2100, dtype=torch.long, device="cuda")
    z[:2099] = -1
    z[2099] = y[1]
    grad, = torch.autograd.grad(lz.token_logprobs(leaf, z).sum(), leaf)
    assert torch.all(grad[:2099] == 0)
    one = torch.ones(1, device="cuda")
    g = grad[2099:]
    assert torch.equal(g, _plain_grad(store.detach()[2099:], y[1:], one, g))


# ---- masks, infinities, NaN ------------------------------------------------------------------------------


@pytest.mark.parametrize("v", [40, 1003, 151552])
@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
def test_masked_vocabulary(dtype, v):
    """-inf and the type's lowest value at masked entries, rows of nothing but one value
    left, rows of the lowest value alone (all entries equal)."""
    low = torch.finfo(dtype).min
    case = _policy_case(8, v, dtype, 3)
    x = case[0]
    x[0, v // 2:] = -math.inf
    x[1, : v // 2] = -math.inf
    x[2, v // 2:] = low
    x[3, :] = -math.inf
    x[3, v // 3] = 1.5
    x[4, :] = low
    x[5, :] = low
    x[5, v - 1] = 2.0
    y = torch.tensor([0, v - 1, 1, v // 3, 2, v - 1, 3, 4], device="cuda")
    lp = oracle.logp64(x, y[:, None], 1.0)[0][:, 0]
    old = lp.float() - 0.1
    _check_policy(x, y, old, case[3], (lp - 0.2).float())
    ids = torch.tensor([0, v - 1, 1, v // 3, 2, v - 1, 3, 4], device="cuda")[:, None].repeat(1, 2)
    ids[:, 1] = -1
    _check_distill(x, ids, torch.zeros(8, 2, device="cuda"))


@pytest.mark.parametrize("v", [40, 32003, 151552])
@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("mask", [-1e6, -1e9, -1e10, -1e20, -3e38])
def test_large_masks(dtype, v, mask):
    """Large finite masks: on half of a row, on all but one entry, on all of it; and rows that are that
    large themselves. What is added to a mask is below its step, so masked entries are equal."""
    x = _logits(8, v, dtype, 3)
    mask = float(torch.tensor(mask, dtype=dtype))
    x[0, : v // 2] = mask
    x[1, v // 2:] = mask
    x[2, :] = mask
    x[2, v // 3] = 1.0
    x[3, :] = mask
    x[4, :] = -mask
    x[5, 1:] = mask
    x[6, :] = mask / 2
    x[6, ::2] = mask
    y = torch.tensor([v - 1, 0, v // 3, 1, 2, 0, 3, 4], device="cuda")
    lp = oracle.logp64(x, y[:, None], 1.0)[0][:, 0]
    adv = torch.ones(8, device="cuda")
    # a row's own large values do not spread its probabilities: only differences from its maximum count
    _check_policy(x, y, lp.float() - 0.1, adv, (lp - 0.2).float())
    ids = torch.stack([y, (y + 7) % v], 1)
    some = torch.tensor([0, 1, 3, 4, 7], device="cuda")  # rows whose list has no entry of probability zero
    ids[:2, 1] = -1
    _check_distill(x[some], ids[some], torch.zeros(5, 2, device="cuda"))


@pytest.mark.parametrize("v", [17, 32003])
def test_tokens_that_are_masked(v):
    """A token of probability zero: -inf as its log-probability, and the gradient's formula."""
    x = _logits(4, v, FP32, 1)
    x[1, 3] = -math.inf
    y = torch.tensor([3, 3, 3, 3], device="cuda")
    leaf = x.requires_grad_(True)
    out = lz.token_logprobs(leaf, y)
    assert out[1] == -math.inf and torch.isfinite(out[[0, 2, 3]]).all()
    grad, = torch.autograd.grad(out, leaf, torch.ones_like(out))
    assert grad[1, 3] == 1 and torch.isfinite(grad).all()


@pytest.mark.parametrize("v", [40, 32003])
@pytest.mark.parametrize("dtype", [BF16, FP32])
def test_infinities_and_nan_stay_in_their_row(v, dtype):
    x = _logits(5, v, dtype, 2)
    x[1, v // 2] = math.inf
    x[2, v // 3] = math.nan
    x[3, :] = -math.inf
    y = torch.zeros(5, dtype=torch.long, device="cuda")
    leaf = x.requires_grad_(True)
    out = lz.token_logprobs(leaf, y)
    assert out.isnan().tolist() == [False, True, True, True, False]
    grad, = torch.autograd.grad(out, leaf, torch.ones_like(out))
    bad = grad.isnan()
    assert not bad[[0, 4]].any() and bad[1:4].all()
    # and rows that do not count are not read
    y = torch.tensor([0, -1, -1, -1, 0], device="cuda")
    z = torch.zeros(5, device="cuda")
    for up in (1.0, 3.0):
        loss = lz.policy_loss(leaf, y, z, z + 1, ref_logp=z, kl_coef=0.1).loss
        grad, = torch.autograd.grad(loss * up, leaf)
        assert torch.isfinite(loss) and torch.isfinite(grad).all() and torch.all(grad[1:4] == 0)
        w = (y >= 0).float()
        loss = lz.distill_loss(leaf, y.clamp(min=0)[:, None], z[:, None].to(dtype), weights=w).loss
        grad, = torch.autograd.grad(loss * up, leaf)
        assert torch.isfinite(loss) and torch.isfinite(grad).all() and torch.all(grad[1:4] == 0)


def test_ids_beyond_the_vocabulary_show():
    x = _logits(4, 100, BF16, 1).requires_grad_(True)
    y = torch.tensor([1, 100, 2**40, 99], device="cuda")
    z = torch.zeros(4, device="cuda")
    out = lz.token_logprobs(x, y)
    assert out.isnan().tolist() == [False, True, True, False]
    grad, = torch.autograd.grad(out, x, torch.ones_like(out))
    assert grad[1:3].isnan().all() and torch.isfinite(grad[[0, 3]]).all()
    out = lz.policy_loss(x, y, z, z + 1)
    assert out.loss.isnan() and out.logp.isnan().tolist() == [False, True, True, False]
    grad, = torch.autograd.grad(out.loss, x)
    assert grad[1:3].isnan().all() and torch.isfinite(grad[[0, 3]]).all()
    ids = torch.stack([torch.zeros_like(y), y], 1)
    for up in (1.0, 2.0):
        out = lz.distill_loss(x, ids, torch.zeros(4, 2, device="cuda"))
        assert out.loss.isnan() and out.kl.isnan().tolist() == [False, True, True, False]
        grad, = torch.autograd.grad(out.loss * up, x)
        assert grad[1:3].isnan().all() and torch.isfinite(grad[[0, 3]]).all()


def test_nothing_counts():
    for v in (50, 32003):
        x = _logits(3, v, BF16, 1).requires_grad_(True)
        y = torch.full((3,), -100, device="cuda")
        z = torch.zeros(3, device="cuda")
        out = lz.policy_loss(x, y, z, z)
        assert out.loss == 0 and torch.all(torch.autograd.grad(out.loss, x)[0] == 0)
        out = lz.policy_loss(x, y + 100, z, z, weights=z)
        assert out.loss == 0 and torch.all(torch.autograd.grad(out.loss, x)[0] == 0)
        out = lz.distill_loss(x, y[:, None], z[:, None])
        assert out.loss == 0 and torch.all(torch.autograd.grad(out.loss * 2, x)[0] == 0)
    x = torch.empty(0, 50, device="cuda", requires_grad=True)  # no rows at all
    e = torch.empty(0, device="cuda")
    for loss in (lz.policy_loss(x, e.long(), e, e).loss, lz.token_logprobs(x, e.long()).sum(),
                 lz.distill_loss(x, e.long().view(0, 3), e.view(0, 3)).loss):
        assert loss == 0
        assert torch.autograd.grad(loss, x)[0].shape == (0, 50)
    x = torch.empty(2, 0, 50, device="cuda", requires_grad=True)
    loss = lz.preference_loss(x, torch.empty(2, 0, dtype=torch.long, device="cuda")).loss
    assert abs(float(loss.detach()) - math.log(2)) < 1e-6
    assert torch.autograd.grad(loss, x)[0].shape == (2, 0, 50)


# ---- what the arguments mean ----------------------------------------------------------------------------


@pytest.mark.parametrize("temperature", [0.05, 0.7, 2.0])
@pytest.mark.parametrize("dtype", [BF16, FP32])
def test_temperature(dtype, temperature):
    _check_policy(*_policy_case(9, 1003, dtype, 5, temperature=temperature), temperature=temperature)
    _check_distill(*_distill_case(9, 1003, 12, dtype, 5), temperature=temperature)


@pytest.mark.parametrize("v", [1003, 64000])
def test_weights_and_denom(v):
    case = _policy_case(30, v, BF16, 6)
    w = torch.rand(30, device="cuda", generator=_gen(2))
    w[torch.rand(30, device="cuda", generator=_gen(3)) < 0.4] = 0
    case[1][4] = -7
    _check_policy(*case, w=w)
    _check_policy(*case, w=w, denom=123.0)
    _check_policy(*case[:4], None, w=(w > 0))
    x, ids, t = _distill_case(30, v, 9, BF16, 6)
    _check_distill(x, ids, t, w=w)
    _check_distill(x, ids, t, w=w, denom=0.5)
    a = lz.policy_loss(*case[:4], weights=w, denom=torch.tensor(3.0, device="cuda")).loss
    assert torch.equal(a, lz.policy_loss(*case[:4], weights=w, denom=3).loss)


def test_duplicate_and_padded_teacher_entries():
    x, ids, t = _distill_case(6, 5000, 40, FP32, 8)
    ids[0, 5] = ids[0, 20]
    ids[1, :] = ids[1, 0]       # one index forty times
    ids[2, 10:] = -1
    ids[3, :] = -1
    ids[4, ::2] = -5
    t[5, :] = -math.inf         # and one entry of weight
    t[5, 7] = 0.0
    _check_distill(x, ids, t)
    x, ids, t = _distill_case(3, 5000, 1024, BF16, 9)
    ids[1, 512:] = ids[1, :512]
    _check_distill(x, ids, t)


@pytest.mark.parametrize("v", [1000, 32003, 151552])
@pytest.mark.parametrize("upstream", [0.125, 1.0, -3.0, 65536.0, 0.0])
def test_upstream(v, upstream):
    """Another upstream than 1 gives the formula's gradient, rounded once."""
    _check_policy(*_policy_case(5, v, BF16, 6), upstream=upstream)
    if abs(upstream) <= 3:
        _check_policy(*_policy_case(5, v, FP16, 6), upstream=upstream)
    _check_distill(*_distill_case(5, v, 9, FP32, 6), upstream=upstream)


def test_backward_twice_and_leaves():
    """A retained graph's second pass writes into other memory; leaves add up."""
    x, y, old, adv, r = _policy_case(20, 4099, BF16, 2)
    x.requires_grad_(True)
    loss = lz.policy_loss(x, y, old, adv, ref_logp=r, kl_coef=0.1).loss
    a, = torch.autograd.grad(loss, x, retain_graph=True)
    b, = torch.autograd.grad(loss, x, retain_graph=True)
    assert torch.equal(a, b) and a.data_ptr() != b.data_ptr()
    loss.backward(retain_graph=True)
    first = x.grad.clone()
    assert torch.equal(first, a)
    loss.backward()
    assert torch.equal(x.grad, (a.float() * 2).bfloat16()) and torch.equal(a, b)
    with pytest.raises(RuntimeError):
        loss.backward()
    loss = lz.policy_loss(x, y, old, adv).loss
    with torch.no_grad():
        x.add_(1)
    with pytest.raises(RuntimeError):  # the logits changed
        loss.backward()


@pytest.mark.parametrize("v", [700, 40000])
def test_what_the_forward_pass_alone_read_may_be_gone(v):
    """The backward pass for another upstream, after the forward pass's weights (converted copies
    here) and scores have been freed and their memory given back."""
    case = _policy_case(12, v, BF16, 3)
    x, ids, t = _distill_case(12, v, 9, BF16, 4)
    mask = torch.rand(12, device="cuda", generator=_gen(1)) < 0.7
    want = [_check_policy(*case, w=mask, upstream=2.0)[1], _check_distill(x, ids, t, w=mask, upstream=2.0)[1]]
    leaves = [case[0].detach().requires_grad_(True), x.detach().requires_grad_(True)]
    losses = [lz.policy_loss(leaves[0], case[1], case[2].clone(), case[3].clone(), ref_logp=case[4].clone(), weights=mask.clone(),
                             clip_low=0.2, clip_high=0.25, kl_coef=0.1).loss,
              lz.distill_loss(leaves[1], ids.clone(), t.clone(), weights=mask.clone()).loss]
    torch.cuda.synchronize()
    torch.cuda.empty_cache()
    for loss, leaf, g in zip(losses, leaves, want):
        assert torch.equal(torch.autograd.grad(loss * 2, leaf)[0], g)


def test_two_threads_on_one_graph():
    import threading

    x, y, old, adv, r = _policy_case(40, 9000, BF16, 2)
    x.requires_grad_(True)
    loss = lz.policy_loss(x, y, old, adv, ref_logp=r, kl_coef=0.1).loss
    want, = torch.autograd.grad(lz.policy_loss(x, y, old, adv, ref_logp=r, kl_coef=0.1).loss * 3, x)
    one, = torch.autograd.grad(lz.policy_loss(x, y, old, adv, ref_logp=r, kl_coef=0.1).loss, x)
    got, errors = [None] * 8, []

    def work(k):
        try:
            up = torch.tensor(3.0 if k % 2 else 1.0, device="cuda")
            got[k], = torch.autograd.grad(loss, x, up, retain_graph=True)
        except Exception as e:  # noqa: BLE001
            errors.append(e)

    threads = [threading.Thread(target=work, args=(k,)) for k in range(8)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert not errors
    for k in range(8):
        assert torch.equal(got[k], want if k % 2 else one)
    assert len({g.data_ptr() for g in got}) == 8


def test_no_second_derivatives():
    """A graph of the gradient may be recorded; to differentiate it is refused."""
    x, y, old, adv, r = _policy_case(6, 300, FP32, 2)
    x.requires_grad_(True)
    ids = y[:, None]
    for f in (lambda: lz.policy_loss(x, y, old, adv).loss, lambda: lz.token_logprobs(x, y).sum(),
              lambda: lz.distill_loss(x, ids, torch.zeros(6, 1, device="cuda")).loss,
              lambda: lz.preference_loss(x.view(2, 3, 300), y.view(2, 3)).loss):
        plain, = torch.autograd.grad(f(), x)
        g, = torch.autograd.grad(f(), x, create_graph=True)
        assert torch.equal(g.detach(), plain)
        with pytest.raises(RuntimeError):
            g.sum().backward()


def test_saved_tensors_may_live_elsewhere():
    x, y, old, adv, r = _policy_case(6, 301, BF16, 2)
    store = torch.zeros(2, 4, 301, device="cuda", dtype=BF16)
    store[:, :3] = x.view(2, 3, 301)
    leaf = store.requires_grad_(True)
    args = [t.view(2, 3) for t in (y, old, adv)]
    want, = torch.autograd.grad(lz.policy_loss(leaf[:, :3], *args).loss * 3, leaf)
    with torch.autograd.graph.save_on_cpu():
        loss = lz.policy_loss(leaf[:, :3], *args).loss * 3
    got, = torch.autograd.grad(loss, leaf)
    assert torch.equal(got, want)


def test_without_gradient_the_same_values():
    x, y, old, adv, r = _policy_case(20, 40000, BF16, 2)
    ids = y[:, None].repeat(1, 3)
    t = torch.randn(20, 3, device="cuda")
    a = lz.policy_loss(x, y, old, adv, ref_logp=r, kl_coef=0.1)
    d = lz.distill_loss(x, ids, t)
    x.requires_grad_(True)
    b = lz.policy_loss(x, y, old, adv, ref_logp=r, kl_coef=0.1)
    e = lz.distill_loss(x, ids, t)
    assert not a.loss.requires_grad and b.loss.requires_grad
    assert not b.logp.requires_grad and not b.kl.requires_grad
    assert torch.equal(a.clipped, b.clipped)
    # the two may add a row up in another order
    off = 2 * oracle.logp_off(x.detach(), 1.0, a.logp.double())
    _near(b.logp, a.logp.double(), off, "logp")
    _near(e.kl, d.kl.double(), off + 1e-6, "kl")


def test_same_bits_each_time():
    for n, v, dtype in ((1, 151552, BF16), (200, 32003, FP16), (50, 151936, FP32), (500, 1000, BF16)):
        case = _policy_case(n, v, dtype, 4)
        ids = torch.randint(0, v, (n, 70), device="cuda", generator=_gen(1))
        t = torch.randn(n, 70, device="cuda", generator=_gen(2))
        runs = []
        for _ in range(3):
            leaf = case[0].detach().requires_grad_(True)
            out = lz.policy_loss(leaf, *case[1:4], ref_logp=case[4], kl_coef=0.1)
            g, = torch.autograd.grad(out.loss, leaf)
            d = lz.distill_loss(leaf, ids, t)
            h, = torch.autograd.grad(d.loss, leaf)
            runs.append((out.loss, out.logp, out.kl, g, d.loss, d.kl, h))
        for other in runs[1:]:
            assert all(torch.equal(a, b) for a, b in zip(runs[0], other))


# ---- streams and graphs ---------------------------------------------------------------------------------


def test_two_streams_at_once():
    cases = [_policy_case(64, 32003, BF16, s) for s in (1, 2)]
    want = []
    for c in cases:
        leaf = c[0].detach().requires_grad_(True)
        out = lz.policy_loss(leaf, *c[1:4], ref_logp=c[4], kl_coef=0.1)
        want.append((out.loss, *torch.autograd.grad(out.loss, leaf)))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    got = [[], []]
    for _ in range(5):
        for k, (s, c) in enumerate(zip(streams, cases)):
            with torch.cuda.stream(s):
                leaf = c[0].detach().requires_grad_(True)
                out = lz.policy_loss(leaf, *c[1:4], ref_logp=c[4], kl_coef=0.1)
                got[k].append((out.loss, *torch.autograd.grad(out.loss, leaf)))
    torch.cuda.synchronize()
    for k in range(2):
        for loss, g in got[k]:
            assert torch.equal(loss, want[k][0]) and torch.equal(g, want[k][1])


@pytest.mark.parametrize("v", [1000, 50021, 151552])
def test_captured_and_replayed(v):
    """Forward and backward in one graph, replayed on other inputs; two graphs share nothing."""
    def step(x, y, old, adv, r, ids, t, scale):
        a = lz.policy_loss(x, y, old, adv, ref_logp=r, kl_coef=0.1)
        d = lz.distill_loss(x, ids, t)
        f = lz.preference_loss(x.view(4, -1, v), y.view(4, -1))
        lp = lz.token_logprobs(x, y)
        grads = [torch.autograd.grad(loss * scale, x)[0] for loss in (a.loss, d.loss, f.loss, lp.sum())]
        return [a.loss, a.logp, a.clipped, d.loss, d.kl, f.loss, f.chosen_rewards, lp, *grads]

    def inputs(seed):
        x, y, old, adv, r = _policy_case(12, v, BF16, seed)
        return [x, y, old, adv, r, torch.randint(0, v, (12, 30), device="cuda", generator=_gen(seed)),
                torch.randn(12, 30, device="cuda", generator=_gen(seed + 1)), torch.ones((), device="cuda")]

    static = [inputs(1), inputs(2)]
    graphs, outs = [], []
    side = torch.cuda.Stream()
    for s in static:
        s[0].requires_grad_(True)
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step(*s)
        torch.cuda.current_stream().wait_stream(side)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            o = step(*s)
        graphs.append(g)
        outs.append(o)
    for round_ in range(2):
        for k in (0, 1):
            new = inputs(10 + 2 * round_ + k)
            new[-1].fill_(1.0 + round_)  # the second time with another upstream
            with torch.no_grad():
                for a, b in zip(static[k], new):
                    a.copy_(b)
            graphs[k].replay()
        for k in (0, 1):
            new = inputs(10 + 2 * round_ + k)
            new[-1].fill_(1.0 + round_)
            new[0].requires_grad_(True)
            for a, b in zip(outs[k], step(*new)):
                assert torch.equal(a, b)
    torch.cuda.synchronize()


def test_a_dropped_graph_frees_its_memory():
    """No cycle holds the gradient that the forward pass wrote, or the logits."""
    import gc

    x, y, old, adv, r = _policy_case(64, 40000, BF16, 2)
    ids = y[:, None]
    t = torch.zeros(64, 1, device="cuda")
    gc.collect()
    gc.disable()
    try:
        for f in (lambda z: lz.policy_loss(z, y, old, adv, ref_logp=r).loss, lambda z: lz.distill_loss(z, ids, t).loss,
                  lambda z: lz.token_logprobs(z, y).sum(),
                  lambda z: lz.preference_loss(z.view(2, 32, -1), y.view(2, 32)).loss):
            before = torch.cuda.memory_allocated()
            leaf = x.clone().requires_grad_(True)
            loss = f(leaf)
            del loss
            loss = f(leaf)
            g, = torch.autograd.grad(loss, leaf)
            del loss, g, leaf
            assert torch.cuda.memory_allocated() == before
    finally:
        gc.enable()


FIRST_CALL = r"""
import torch
import results_b200 as lz
x = torch.randn(6, 50000, device="cuda", dtype=torch.bfloat16).requires_grad_(True)
small = torch.randn(6, 500, device="cuda").requires_grad_(True)
y = torch.arange(6, device="cuda")
z = torch.zeros(6, device="cuda")
out, g = [], torch.cuda.CUDAGraph()
from results_b200 import _native
_native.cuda()
with torch.cuda.graph(g):
    for t in (x, small):
        out += torch.autograd.grad(lz.policy_loss(t, y, z - 9, z + 1).loss, t)
        out += torch.autograd.grad(lz.token_logprobs(t, y), t, z + 1)
g.replay()
torch.cuda.synchronize()
for i, t in enumerate((x, small)):
    assert torch.equal(out[2 * i], torch.autograd.grad(lz.policy_loss(t, y, z - 9, z + 1).loss, t)[0])
    assert torch.equal(out[2 * i + 1], torch.autograd.grad(lz.token_logprobs(t, y), t, z + 1)[0])
print("captured first ok")
"""


def test_first_call_of_a_process_is_captured():
    import os
    import subprocess
    import sys

    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, "-c", FIRST_CALL], cwd=root, capture_output=True, text=True, timeout=300)
    assert "captured first ok" in r.stdout, r.stdout + r.stderr


def test_many_rows_of_every_kind():
    """More rows than teams and clusters, some of which do not count, at sizes where the kernels change."""
    for n, v, dtype in ((9000, 700, BF16), (5000, 8000, FP16), (1300, 9001, FP32), (400, 30011, FP16), (311, 60000, BF16),
                        (2500, 24000, BF16), (300, 33000, FP32), (700, 70000, BF16)):
        case = _policy_case(n, v, dtype, n)
        case[1][torch.rand(n, device="cuda", generator=_gen(1)) < 0.3] = -1
        w = torch.rand(n, device="cuda", generator=_gen(2))
        w[torch.rand(n, device="cuda", generator=_gen(3)) < 0.3] = 0
        _check_policy(*case, w=w, upstream=1.0)
        _check_policy(*case, w=w, upstream=-0.5)
        x, ids, t = _distill_case(n, v, 33, dtype, n)
        ids[::7, 5:] = -1
        _check_distill(x, ids, t, w=w)
        _check_distill(x, ids, t, w=w, upstream=2.0)
        del case, x


@pytest.mark.parametrize("n,v,dtype", [(150001, 8, BF16), (40003, 33, FP16), (20000, 41, FP32), (15000, 1001, BF16),
                                       (14500, 512, FP32), (14209, 1024, FP16), (5001, 2047, FP16), (9999, 1022, FP32)])
def test_very_many_short_rows(n, v, dtype):
    """Rows that a part of a warp has, several at once: ragged batches, rows that do not count in
    every place, weights, masked entries, rows of huge masks only, and both ways of a gradient."""
    x, y, old, adv, ref = _policy_case(n, v, dtype, n)
    big = 6e4 if dtype is FP16 else 1e10
    x[7::50] = -big
    x[11::13, v // 2] = -math.inf
    y = torch.where(y == v // 2, 0, y)
    y[11::13] = torch.where(y[11::13] == v // 2, 0, y[11::13])
    lp = oracle.logp64(x, y[:, None], 1.0)[0][:, 0]
    old, ref = (lp - 0.1 * (old * 7).sin()).float(), (lp + 0.3 * (ref * 5).sin()).float()
    y[::9] = -1
    y[n // 3:n // 3 + 70] = -1
    y[-3:] = -1
    w = torch.rand(n, device="cuda", generator=_gen(2)) + 0.5
    w[5::17] = 0
    _check_policy(x, y, old, adv, ref, w)
    _check_policy(x, y.int(), old, adv, ref, w, upstream=0.5, denom=77.0)
    test_token_logprobs_sizes(n, v, dtype)


@pytest.mark.parametrize("ids", [torch.int64, torch.int32])
def test_many_rows_in_order(ids):
    """More rows than one block sorts, streamed: runs that do not count at either end and in between."""
    n, v = 3001, 24000
    x, y, old, adv, ref = _policy_case(n, v, BF16, 4)
    y[:700], y[1300:1600], y[2990:], y[::11] = -1, -1, -1, -1
    w = torch.rand(n, device="cuda", generator=_gen(2)) + 0.5
    w[3::19] = 0
    _check_policy(x, y.to(ids), old, adv, ref, w)
    _check_policy(x, y.to(ids), old, adv, ref, None, upstream=0.5)
    x, idx, t = _distill_case(n, 52000, 20, BF16, 3)
    _check_distill(x, idx.to(ids), t, w)
    _check_distill(x, idx.to(ids), t, torch.zeros_like(w))


def test_losses_under_autocast_and_checkpoint():
    from torch.utils.checkpoint import checkpoint

    w = (torch.randn(500, 64, device="cuda", generator=_gen(1)) * 0.2).requires_grad_(True)
    h = torch.randn(12, 64, device="cuda", generator=_gen(2))
    y = _tokens(12, 500, 3)
    with torch.autocast("cuda", dtype=BF16):
        logits = h @ w.t()
        assert logits.dtype == BF16
        loss = -lz.token_logprobs(logits, y).mean()
    a, = torch.autograd.grad(loss, w)
    z = torch.zeros(12, device="cuda")

    def f(w):
        return lz.policy_loss((h @ w.t()).bfloat16(), y, z, z + 1).loss

    b, = torch.autograd.grad(f(w), w)
    c, = torch.autograd.grad(checkpoint(f, w, use_reentrant=False), w)
    assert torch.isfinite(a).all() and torch.equal(b, c)


def test_a_training_run_of_all():
    """A rollout scored, a policy step on its scores, a preference step and a distillation
    step of a small head: each output feeds the next, and the head's gradient is the formula's."""
    v, n, h = 1000, 32, 48
    head = (torch.randn(v, h, device="cuda", generator=_gen(1)) * 0.3)
    x = torch.randn(n, h, device="cuda", generator=_gen(2))
    with torch.no_grad():
        logits = x @ head.t()
        y = _tokens(n, v, 3, logits)
        old = lz.token_logprobs(logits, y)
    w = head.clone().requires_grad_(True)
    adv = torch.randn(n, device="cuda", generator=_gen(4))

    def head_off(want, off, slope_off):  # the product's: n terms of fp32, each rounded, the sum too
        bound = oracle.grad_off(want, FP32, off, slope_off)
        return bound.t() @ x.double().abs() + (n + 2) * 2.0 ** -23 * (want["grad"].abs().t() @ x.double().abs())

    assert not torch.backends.cuda.matmul.allow_tf32
    for _ in range(2):
        logits = x @ w.t()
        out = lz.policy_loss(logits, y, old, adv, ref_logp=old, kl_coef=0.05)
        g, = torch.autograd.grad(out.loss, w)
        want = oracle.policy(logits.detach(), y, old, adv, old, None, 0.2, 0.2, 0.05, 1.0, None)
        off = oracle.logp_off(logits.detach(), 1.0, want["logp"])
        _near(g, want["grad"].t() @ x.double(), head_off(want, off, want["bend"] * off), "policy")
        with torch.no_grad():
            w -= 0.05 * g
        old = out.logp
    logits = x @ w.t()
    out = lz.preference_loss(logits.view(8, 4, v), y.view(8, 4), ref_logp=old.view(8, 4).sum(1))
    g, = torch.autograd.grad(out.loss, w)
    ends = list(range(0, 33, 4))
    want = oracle.preference(logits.detach(), y, old.view(8, 4).sum(1), ends, 0.1, 0.0, False, 1.0)
    off = oracle.logp_off(logits.detach(), 1.0, want["logp"])
    slope_off = 0.1 / 4 / 4 * (8 * 0.1 * off.max() + 2.0 ** -22) + 2.0 ** -23 * want["slope"].abs()
    _near(g, want["grad"].t() @ x.double(), head_off(want, off, slope_off), "preference")
    top = (x @ head.t()).topk(16)
    out = lz.distill_loss(x @ w.t(), top.indices, top.values)
    g, = torch.autograd.grad(out.loss, w)
    want = oracle.distill((x @ w.t()).detach(), top.indices, top.values, None, 1.0, None)
    q_off = 2.0 ** -24 * (17 + 4 * top.values.abs().amax(1).double()) * want["slope"].abs()
    extra = q_off.max() * x.double().abs().sum(0)  # of each entry of the list, wherever it stands
    _near(g, want["grad"].t() @ x.double(), head_off(want, off, torch.zeros_like(off)) + extra, "distill")
