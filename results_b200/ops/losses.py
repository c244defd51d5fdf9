"""Losses over the vocabulary: what an RL trainer, a preference trainer or a
student computes between its output head and its backward pass.

    logp = token_logprobs(logits, tokens)                      # rollout / reference log-probabilities
    out = policy_loss(logits, tokens, old_logp, advantages, ref_logp=ref, kl_coef=0.02)
    out = preference_loss(logits, tokens, ref_logp=ref)        # first half chosen, second half rejected
    out = distill_loss(logits, teacher_ids, teacher_logits)    # the teacher's top entries
    out.loss.backward()

``logits`` is ``[..., vocab]`` in bf16, fp16 or fp32, ``tokens`` its leading
shape in int32 or int64. Leading dimensions may have any strides (``logits[:, :-1]``
is read in place; gradients are fastest where rows start at the same offset from
a 16-byte border as in a contiguous tensor); a vocabulary that is not contiguous
is copied. A negative token marks a row that does not count (prompt, padding):
its logits are not read, its outputs and its gradient are zero. The same holds
for rows of weight zero. A token or teacher id beyond the vocabulary, or NaN or
+inf among a teacher's entries, makes a row that counts (and the loss) NaN.

Sums and log-probabilities are held in 32 bits or more and a gradient is
rounded once, to the logits' type. Results do not depend on timing: the same
inputs give the same bits.

On the GPU ``policy_loss`` and ``distill_loss`` write the gradient during the
forward pass, while a row is still on the chip, for an upstream gradient of 1;
the backward pass looks at the upstream on the device and computes the
gradient anew, from the logits, if it is another (a loss divided by the number
of micro batches, a loss scaler). Pass such a factor through ``denom`` instead
to keep the cheaper way, and capture both passes into one CUDA graph: a backward
pass captured apart computes the gradient anew at every replay. The logits must
not be changed before the backward pass. CUDA tensors run the kernels in
csrc/lz_losses.cu on the current stream of their device, with a first derivative
in the logits by the backward pass (no second one, no forward mode, no tracing;
inside a function that torch.compile takes they run as they are);
CPU tensors run the definitions in 64-bit torch operations.
"""
from __future__ import annotations

import ctypes as C
import math
from typing import NamedTuple

import torch
from torch.autograd import forward_ad

from .. import _native, _native_sigs
from ..utils.dtypes import LZ_BF16, LZ_F16, LZ_F32
from ..utils.trace import traced

LOGP, POLICY, DISTILL = 0, 1, 2
_NAMES = ("token log-probabilities", "policy loss", "distillation loss")
MAX_TOP = 1024
_HEAD, _PER_ROW = 2, 5  # doubles of the workspace (csrc/lz_losses.h)
_DTYPES = {torch.float32: LZ_F32, torch.float16: LZ_F16, torch.bfloat16: LZ_BF16}
_IDS = (torch.int64, torch.int32)

_p, _l, _f, _d, _i = C.c_void_p, C.c_longlong, C.c_float, C.c_double, C.c_int


class _LossArgs(C.Structure):  # struct LzLossArgs
    _fields_ = [("logits", _p), ("outer_stride", _l), ("inner_stride", _l), ("inner", _l), ("rows", _l), ("vocab", _l),
                ("grad", _p), ("ids", _p), ("teacher", _p), ("old_logp", _p), ("advantages", _p), ("ref_logp", _p),
                ("weights", _p), ("denom_ptr", _p), ("upstream", _p), ("row_upstream", _p), ("loss", _p), ("logp", _p),
                ("kl", _p), ("clipped", _p), ("work", _p), ("denom", _d), ("inv_temperature", _f), ("clip_low", _f),
                ("clip_high", _f), ("kl_coef", _f), ("kind", _i), ("dtype", _i), ("ids64", _i), ("top", _i),
                ("teacher_dtype", _i), ("device", _i), ("fresh", _i), ("capture", C.c_ulonglong),
                ("wait_ns", C.c_ulonglong)]


class _PairArgs(C.Structure):  # struct LzPairArgs
    _fields_ = [("logp_work", _p), ("ids", _p), ("offsets", _p), ("ref_logp", _p), ("loss", _p),
                ("rewards", _p), ("work", _p), ("rows", _l), ("pairs", _l), ("length", _l), ("beta", _d), ("smoothing", _d),
                ("normalized", _i), ("ids64", _i), ("offsets64", _i), ("device", _i)]


_native_sigs.add_cuda({
    "lz_loss_forward": (_i, C.POINTER(_LossArgs), _p),
    "lz_loss_backward": (_i, C.POINTER(_LossArgs), _p),
    "lz_loss_pairs": (_i, C.POINTER(_PairArgs), _p),
})


class PolicyLoss(NamedTuple):
    loss: torch.Tensor            # scalar
    logp: torch.Tensor            # per token, no gradient
    kl: torch.Tensor | None       # per token, no gradient; None without ref_logp
    clipped: torch.Tensor         # per token: the clip is active


class PreferenceLoss(NamedTuple):
    loss: torch.Tensor              # scalar
    chosen_rewards: torch.Tensor    # per pair: beta (sum of logp - ref), no gradient
    rejected_rewards: torch.Tensor


class DistillLoss(NamedTuple):
    loss: torch.Tensor  # scalar
    kl: torch.Tensor    # per row, no gradient


# ---- checks ---------------------------------------------------------------------------------------------


def _check_logits(what: str, logits: torch.Tensor) -> None:
    if logits.dtype not in _DTYPES:
        raise TypeError(f"{what}: logits are {logits.dtype}; expected bfloat16, float16 or float32")
    if not logits.dim() or not 0 < logits.shape[-1] < 2**31:
        raise ValueError(f"{what}: logits of shape {tuple(logits.shape)}; expected a vocabulary of 1 to 2^31 - 1 entries")
    if not (logits.is_cuda or logits.is_cpu):
        raise ValueError(f"{what}: device {logits.device} is not supported")


def _check_ids(what: str, name: str, ids: torch.Tensor, shape, device) -> torch.Tensor:
    if ids.dtype not in _IDS:
        raise TypeError(f"{what}: {name} are {ids.dtype}; expected int64 or int32")
    if ids.shape != shape:
        raise ValueError(f"{what}: {name} have shape {tuple(ids.shape)}; expected {tuple(shape)}")
    if ids.device != device:
        raise ValueError(f"{what}: {name} are on {ids.device}, the logits on {device}")
    return ids.contiguous()


def _check_rows(what: str, name: str, t: torch.Tensor | None, shape, device, any_type=False) -> torch.Tensor | None:
    """A value per row (or sequence) as contiguous fp32."""
    if t is None:
        return None
    if t.dtype is torch.float32 and t.shape == shape and t.device == device and not t.requires_grad:
        return t.contiguous()
    if not (t.is_floating_point() or any_type) or t.is_complex():
        raise TypeError(f"{what}: {name} is {t.dtype}; expected a floating-point type")
    if t.shape != shape:
        raise ValueError(f"{what}: {name} has shape {tuple(t.shape)}; expected {tuple(shape)}")
    if t.device != device:
        raise ValueError(f"{what}: {name} is on {t.device}, the logits on {device}")
    if t.requires_grad:
        raise ValueError(f"{what}: {name} requires a gradient, and this loss gives none to it; detach it")
    return t.to(torch.float32).contiguous()


def _check_number(what: str, name: str, v, low: float, high: float = math.inf, open_low: bool = False) -> float:
    v = float(v)
    if not (v > low if open_low else v >= low) or v > high or math.isinf(v):
        raise ValueError(f"{what}: {name} = {v} is out of range")
    return v


def _check_temperature(what: str, temperature) -> float:
    t = _check_number(what, "temperature", temperature, 0.0, open_low=True)
    if not 1e-6 <= t <= 1e6:
        raise ValueError(f"{what}: temperature = {t} is out of range")
    return t


def _check_denom(what: str, denom, device):
    """None, a positive number, or a tensor of one value on the logits' device."""
    if denom is None or not isinstance(denom, torch.Tensor):
        return None if denom is None else _check_number(what, "denom", denom, 0.0, open_low=True)
    if denom.numel() != 1 or denom.is_complex():
        raise ValueError(f"{what}: denom has shape {tuple(denom.shape)}; expected one number")
    if denom.device != device:
        raise ValueError(f"{what}: denom is on {denom.device}, the logits on {device}")
    if denom.requires_grad:
        raise ValueError(f"{what}: denom requires a gradient, and this loss gives none to it; detach it")
    return denom.to(torch.float32)


def _check_modes(what: str, *tensors: torch.Tensor | None) -> None:
    """CUDA tensors: what goes past autograd functions would be lost in the kernels."""
    if _is_tracing():
        raise RuntimeError(f"{what}: a call with CUDA tensors cannot be traced")
    for t in tensors:
        if isinstance(t, torch.Tensor) and forward_ad.unpack_dual(t).tangent is not None:
            raise RuntimeError(f"{what}: no forward-mode derivative for CUDA tensors")


# ---- native calls ---------------------------------------------------------------------------------------
#
# Small calls are bound by what runs on the host: the arguments are built in one
# go, the backward pass takes the forward pass's, and only the differentiable
# output goes through autograd.


def _ptr(t: torch.Tensor | None):
    return None if t is None else t.data_ptr()


def _rows_of(x: torch.Tensor):
    """(tensor, outer stride, inner stride, inner, rows): row r starts at
    (r // inner) * outer stride + (r % inner) * inner stride. Copies only where
    two strides and a contiguous vocabulary cannot say it."""
    v = x.shape[-1]
    if x.is_contiguous():
        rows = x.numel() // v
        return x, 0, v, rows or 1, rows
    lead = x.shape[:-1]
    if x.stride(-1) != 1 and v > 1 or len(lead) > 2:
        return _rows_of(x.contiguous())
    if len(lead) == 2:
        return x, x.stride(0), x.stride(1), max(1, lead[1]), lead[0] * lead[1]
    return x, 0, x.stride(0) if lead else 0, max(1, math.prod(lead)), math.prod(lead)


_lib = None
_saved_hooks = torch._C._autograd._top_saved_tensors_default_hooks
_is_tracing = torch._C._is_tracing

def _as_it_is() -> None:
    """A function that begins with this is run by torch.compile as it is: it raises while the compiler traces it."""
    if torch.compiler.is_dynamo_compiling():
        raise RuntimeError("native calls are not compiled")


_APART = 1  # LZ_LOSS_APART


def _launch(fn: str, a) -> bool:
    """False: nothing ran, the forward pass belongs to another graph capture."""
    global _lib
    _as_it_is()
    if _lib is None:
        _lib = _native.cuda()
    rc = getattr(_lib, fn)(C.byref(a), torch._C._cuda_getCurrentRawStream(a.device))
    if rc and rc != _APART:
        _native.check(rc, "preference loss" if fn == "lz_loss_pairs" else _NAMES[a.kind])
    return not rc


class _Call:
    """One call: its arguments, its output `out`, and the tensors that the
    backward pass reads (`keep`, until autograd has them)."""

    def __init__(self, kind, logits, ids, temperature, out, logp=None, kl=None, clipped=None,
                 rows=None, teacher=None, denom=None, numbers=(0.0, 0.0, 0.0), fused=False):
        _as_it_is()
        x, outer_stride, inner_stride, inner, n = _rows_of(logits)
        dev = x.device
        work = torch.empty(_HEAD + _PER_ROW * n, dtype=torch.float64, device=dev)
        # the gradient for upstream 1, written by the forward pass; the first backward pass takes it away
        self.grad = torch.empty_like(logits, memory_format=torch.contiguous_format) if fused else None
        self.out, self.shape = out, logits.shape
        self.keep = (x, ids, work) if teacher is None else (x, ids, work, teacher)
        at = self.at = x.data_ptr(), ids.data_ptr(), work.data_ptr()
        self.strides = x.stride() if outer_stride or inner_stride != x.shape[-1] else None  # None: contiguous
        a = self.args = _LossArgs(at[0], outer_stride, inner_stride, inner, n, x.shape[-1], _ptr(self.grad), at[1])
        a.work, a.inv_temperature, a.kind = at[2], 1.0 / temperature, kind
        a.dtype, a.ids64, a.device = _DTYPES[x.dtype], ids.dtype is torch.int64, dev.index
        a.logp = _ptr(logp)
        if kind == LOGP:
            return
        old, adv, ref, weights = rows
        a.loss, a.kl, a.clipped, a.weights = out.data_ptr(), _ptr(kl), _ptr(clipped), _ptr(weights)
        if isinstance(denom, torch.Tensor):
            a.denom_ptr = denom.data_ptr()
        else:
            a.denom = -1.0 if denom is None else denom
        if kind == POLICY:
            a.old_logp, a.advantages, a.ref_logp = old.data_ptr(), adv.data_ptr(), _ptr(ref)
            a.clip_low, a.clip_high, a.kl_coef = numbers
        else:
            a.teacher, a.teacher_dtype, a.top = teacher.data_ptr(), _DTYPES[teacher.dtype], ids.shape[-1]

    def forward(self) -> None:
        _launch("lz_loss_forward", self.args)

    def set_upstream(self, a, g: int, saved) -> None:
        """`g`: address of the upstream gradient, of each row's log-probability or of the loss."""
        if a.kind == LOGP:
            a.row_upstream = g
        else:
            a.upstream = g

    def backward(self, saved, g) -> torch.Tensor:
        """The gradient is handed out once: a second pass over a retained graph
        writes into memory of its own, and so does a pass that was captured
        apart from the forward pass."""
        _as_it_is()
        a, x = _LossArgs.from_buffer_copy(self.args), saved[0]  # other threads may be here too
        grad = self.__dict__.pop("grad", None)
        if g.dtype is not torch.float32 or not g.is_contiguous():
            g = g.to(torch.float32).contiguous()
        if self.hooked or (x.data_ptr(), saved[1].data_ptr(), saved[2].data_ptr()) != self.at or \
                not (x.is_contiguous() if self.strides is None else x.stride() == self.strides) or \
                (a.kind == DISTILL and saved[3].data_ptr() != a.teacher):
            saved = self.came_back(a, saved)
            x = saved[0]
        self.set_upstream(a, g.data_ptr(), saved)
        if grad is None or not _launch("lz_loss_backward", a):
            a.fresh = 1
            grad = torch.empty(self.shape, dtype=x.dtype, device=x.device)
            a.grad = grad.data_ptr()
            _launch("lz_loss_backward", a)
        return grad

    def came_back(self, a, saved):
        """Hooks on saved tensors may give back other ones, in other layouts, at any address:
        those that the kernels read, with their addresses and strides in `a`."""
        expected = [(a.dtype, a.rows * a.vocab), (torch.int64 if a.ids64 else torch.int32, a.rows * max(1, a.top)),
                    (torch.float64, _HEAD + _PER_ROW * a.rows)]
        if a.kind == DISTILL:
            expected.append((a.teacher_dtype, a.rows * a.top))
        for t, (dtype, n) in zip(saved, expected):
            if t.get_device() != a.device or _DTYPES.get(t.dtype, t.dtype) != dtype or t.numel() != n:
                raise RuntimeError(f"{_NAMES[a.kind]}: a saved tensor came back as {t.dtype} {tuple(t.shape)} on {t.device}")
        x, a.outer_stride, a.inner_stride, a.inner, _ = _rows_of(saved[0].view(self.shape))
        saved = [x, *(t.contiguous() for t in saved[1:])]
        if saved[2].data_ptr() % 16:
            saved[2] = saved[2].clone()
        a.logits, a.ids, a.work = (t.data_ptr() for t in saved[:3])
        if a.kind == DISTILL:
            a.teacher = saved[3].data_ptr()
        return saved


class _Loss(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, call):
        call.forward()
        ctx.save_for_backward(*call.keep)
        call.hooked = _saved_hooks(True) is not None
        ctx.call, out = call, call.out
        call.keep = call.out = None  # the output leads here: it may not be held from here
        return out

    @staticmethod
    def backward(ctx, g):
        if torch.is_grad_enabled():  # a graph of the gradient is recorded: it may not be differentiated itself
            return torch.autograd.function.once_differentiable(_Loss.gradient)(ctx, g), None
        return _Loss.gradient(ctx, g), None

    @staticmethod
    def gradient(ctx, g):
        return ctx.call.backward(ctx.saved_tensors, g)


def _run(call: _Call, logits: torch.Tensor, needs_grad: bool) -> torch.Tensor:
    if needs_grad:
        return _Loss.apply(logits, call)
    call.forward()
    return call.out


class _PairsCall(_Call):
    """The log-probabilities and, from them, the preference loss."""

    def __init__(self, logits, tokens, ref, offsets, p):
        _as_it_is()
        dev, rows, pairs = logits.device, tokens.numel(), p["pairs"]
        logp = torch.empty(tokens.shape, dtype=torch.float32, device=dev)
        super().__init__(LOGP, logits, tokens, p["temperature"], logp, logp)
        self.out = logp.new_empty(())
        self.rewards = logp.new_empty(2 * pairs)
        work = torch.empty(1 + pairs + (rows + 1) // 2, dtype=torch.float64, device=dev)
        self.slopes = 8 * (1 + pairs)  # where the rows' slopes are in it, in bytes
        self.pairs = _PairArgs(
            self.args.work, tokens.data_ptr(), _ptr(offsets), _ptr(ref), self.out.data_ptr(), self.rewards.data_ptr(),
            work.data_ptr(), rows, pairs, p["length"], p["beta"], p["label_smoothing"], p["length_normalized"],
            tokens.dtype is torch.int64, offsets is not None and offsets.dtype is torch.int64, dev.index)
        self.alive = logp, ref, offsets
        self.keep += (work,)

    def forward(self) -> None:
        super().forward()
        _launch("lz_loss_pairs", self.pairs)
        self.alive = None

    def came_back(self, a, saved):
        work = saved[3].contiguous()
        if work.get_device() != a.device or work.dtype is not torch.float64 or work.numel() * 8 < self.slopes + 4 * a.rows:
            raise RuntimeError(f"preference loss: a saved tensor came back as {work.dtype} {tuple(work.shape)} on {work.device}")
        return [*super().came_back(a, saved[:3]), work]

    def set_upstream(self, a, g: int, saved) -> None:
        a.upstream, a.row_upstream = g, saved[3].data_ptr() + self.slopes


# ---- the definitions (CPU tensors) -----------------------------------------------------------------------


def _cpu_nan_rows(x, bad):
    """x [rows], NaN where `bad`, and its gradient there as well, unless the row has no upstream."""
    if x.requires_grad and bool(bad.any()):
        x.register_hook(lambda g: torch.where(bad & (g != 0), math.nan, g))
    return x + torch.where(bad, math.nan, 0.0)


def _cpu_logp(logits, ids, counted, temperature):
    """Log-probabilities of ids [rows, k] in 64 bits; rows that do not count are not looked at."""
    v = logits.shape[-1]
    z = torch.where(counted[:, None], logits.reshape(-1, v).double(), 0.0) / temperature
    return torch.log_softmax(z, -1).gather(1, ids.clamp(0, v - 1).long())


def _cpu_token_logp(logits, y, counted, temperature):
    """Log-probabilities of tokens [rows], zero where a row does not count."""
    logp = _cpu_nan_rows(_cpu_logp(logits, y[:, None], counted, temperature)[:, 0], counted & (y >= logits.shape[-1]))
    return torch.where(counted, logp, 0.0)


def _cpu_scale(weights, counted, denom):
    w = counted.double() if weights is None else torch.where(counted, weights.reshape(-1).double(), 0.0)
    d = w.sum() if denom is None else torch.as_tensor(denom, dtype=torch.float64, device=w.device).reshape(())
    return torch.where(d <= 0, 0.0, w / d)


def _cpu_token_logprobs(logits, tokens, temperature):
    y = tokens.reshape(-1)
    return _cpu_token_logp(logits, y, y >= 0, temperature).float().view(tokens.shape)


def _cpu_policy_loss(logits, tokens, rows, p):
    old, adv, ref, weights = (None if t is None else t.reshape(-1).double() for t in rows)
    y = tokens.reshape(-1)
    scale = _cpu_scale(weights, y >= 0, p["denom"])
    counted = (y >= 0) & (weights != 0) if weights is not None else y >= 0
    logp = _cpu_token_logp(logits, y, counted, p["temperature"])
    ratio = torch.where(counted, logp - old, 0.0).exp()
    low, high = 1.0 - p["clip_low"], 1.0 + p["clip_high"]
    clipped = (((adv > 0) & (ratio > high)) | ((adv < 0) & (ratio < low))) & counted
    each = -adv * torch.where(clipped, torch.where(adv > 0, high, low), ratio)
    kl = None
    if ref is not None:
        d = torch.where(counted, ref - logp, 0.0)
        kl = d.expm1() - d.clamp(max=torch.finfo(torch.float64).max)  # +inf where the token has probability zero
        if p["kl_coef"]:  # 0: watched alone, it may be infinite
            each = each + p["kl_coef"] * kl
        kl = kl.detach().float().view(tokens.shape)
    loss = torch.where(counted, each * scale, 0.0).sum().float()
    return loss, logp.detach().float().view(tokens.shape), kl, clipped.view(tokens.shape)


def _cpu_distill_loss(logits, ids, teacher, weights, p):
    n, k = math.prod(ids.shape[:-1]), ids.shape[-1]
    ids, t = ids.reshape(n, k), teacher.reshape(n, k).double() / p["temperature"]
    there = ids >= 0
    t = torch.where(there, t, -math.inf)
    counted = torch.ones(n, dtype=torch.bool, device=logits.device) if weights is None else weights.reshape(-1) != 0
    some = t.amax(1) != -math.inf
    logq = torch.log_softmax(torch.where(some[:, None], t, 0.0), 1)
    q = torch.where(there & some[:, None], logq.exp(), 0.0)
    bad = (q.isnan() | (ids >= logits.shape[-1])).any(1) & counted
    q, logq = torch.where(bad[:, None], 1.0, q), torch.where(bad[:, None], 0.0, logq)
    logp = _cpu_logp(logits, ids, counted & some, p["temperature"])
    kl = _cpu_nan_rows(torch.where(q > 0, q * (logq - logp), 0.0).sum(1), bad)
    kl = torch.where(counted, kl, 0.0)
    loss = (kl * _cpu_scale(weights, torch.ones_like(counted), p["denom"])).sum().float()
    return loss, kl.detach().float().view(logits.shape[:-1])


def _cpu_preference_loss(logits, tokens, ref, offsets, p):
    y, pairs = tokens.reshape(-1), p["pairs"]
    logp = _cpu_token_logp(logits, y, y >= 0, p["temperature"])
    ends = [s * p["length"] for s in range(2 * pairs + 1)] if offsets is None else offsets.tolist()
    sums = []
    for a, b in zip(ends, ends[1:]):
        if not 0 <= a <= b <= y.numel():
            sums.append(logp.new_tensor(math.nan))
            continue
        count = max(1, int((y[a:b] >= 0).sum())) if p["length_normalized"] else 1
        sums.append(logp[a:b].sum() / count)
    r = p["beta"] * (torch.stack(sums) - (0.0 if ref is None else ref.double()))
    h, eps = r[:pairs] - r[pairs:], p["label_smoothing"]
    # a term of weight zero is none, though an answer that cannot be makes it infinite
    terms = [-w * torch.nn.functional.logsigmoid(x) for w, x in ((1 - eps, h), (eps, -h)) if w]
    return sum(terms).mean().float(), r.detach().float()


# ---- public entry points ---------------------------------------------------------------------------------


def _needs_grad(logits: torch.Tensor) -> bool:
    return logits.requires_grad and torch.is_grad_enabled()


@traced("token_logprobs")
def token_logprobs(logits: torch.Tensor, tokens: torch.Tensor, *, temperature: float = 1.0) -> torch.Tensor:
    """log softmax(logits / temperature) at ``tokens``, fp32, differentiable in the logits."""
    what = "token_logprobs"
    _check_logits(what, logits)
    tokens = _check_ids(what, "tokens", tokens, logits.shape[:-1], logits.device)
    temperature = _check_temperature(what, temperature)
    if not logits.is_cuda:
        return _cpu_token_logprobs(logits, tokens, temperature)
    if _is_tracing() or forward_ad._current_level >= 0:
        _check_modes(what, logits)
    logp = torch.empty(tokens.shape, dtype=torch.float32, device=logits.device)
    return _run(_Call(LOGP, logits, tokens, temperature, logp, logp), logits, _needs_grad(logits))


@traced("policy_loss")
def policy_loss(logits: torch.Tensor, tokens: torch.Tensor, old_logp: torch.Tensor, advantages: torch.Tensor, *,
                ref_logp: torch.Tensor | None = None, weights: torch.Tensor | None = None, clip_low: float = 0.2,
                clip_high: float = 0.2, kl_coef: float = 0.0, temperature: float = 1.0, denom=None) -> PolicyLoss:
    """Clipped policy loss with a KL term to a reference policy:

        ratio = exp(logp - old_logp)
        each  = -min(ratio A, clip(ratio, 1 - clip_low, 1 + clip_high) A) + kl_coef kl
        kl    = exp(ref_logp - logp) - (ref_logp - logp) - 1
        loss  = sum(weights each) / denom

    ``old_logp``, ``advantages``, ``ref_logp`` and ``weights`` (a mask or
    factors) have the tokens' shape. With ``kl_coef`` 0 the KL is an output alone. ``denom`` is a number or a one-element
    tensor on the device (the token count over all micro batches or ranks);
    without it, the sum of the weights of the rows that count. Where that is
    not positive, loss and gradient are zero."""
    what, dev, shape = "policy_loss", logits.device, logits.shape[:-1]
    _check_logits(what, logits)
    tokens = _check_ids(what, "tokens", tokens, shape, dev)
    if ref_logp is None and kl_coef:
        raise ValueError("policy_loss: kl_coef without ref_logp")
    rows = (_check_rows(what, "old_logp", old_logp, shape, dev), _check_rows(what, "advantages", advantages, shape, dev),
            _check_rows(what, "ref_logp", ref_logp, shape, dev),
            _check_rows(what, "weights", weights, shape, dev, any_type=True))
    if rows[0] is None or rows[1] is None:
        raise ValueError("policy_loss: old_logp and advantages are needed")
    p = {"clip_low": _check_number(what, "clip_low", clip_low, 0.0, 1.0),
         "clip_high": _check_number(what, "clip_high", clip_high, 0.0),
         "kl_coef": _check_number(what, "kl_coef", kl_coef, 0.0),
         "temperature": _check_temperature(what, temperature), "denom": _check_denom(what, denom, dev)}
    if not logits.is_cuda:
        return PolicyLoss(*_cpu_policy_loss(logits, tokens, rows, p))
    if _is_tracing() or forward_ad._current_level >= 0:
        _check_modes(what, logits, old_logp, advantages, ref_logp, weights, denom)
    needs_grad, old = _needs_grad(logits), rows[0]  # old_logp: contiguous, fp32, of the tokens' shape
    logp, clipped = torch.empty_like(old), torch.empty_like(old, dtype=torch.bool)
    kl = None if ref_logp is None else torch.empty_like(old)
    call = _Call(POLICY, logits, tokens, p["temperature"], old.new_empty(()), logp, kl, clipped, rows, None, p["denom"],
                 (p["clip_low"], p["clip_high"], p["kl_coef"]), needs_grad)
    return PolicyLoss(_run(call, logits, needs_grad), logp, kl, clipped)


@traced("preference_loss")
def preference_loss(logits: torch.Tensor, tokens: torch.Tensor, *, ref_logp: torch.Tensor | None = None,
                    cu_seqlens: torch.Tensor | None = None, beta: float = 0.1, label_smoothing: float = 0.0,
                    length_normalized: bool = False, temperature: float = 1.0) -> PreferenceLoss:
    """Preference loss on paired log ratios. The batch holds 2 P sequences, the
    P chosen ones first, then their rejected partners in the same order:
    ``logits`` ``[2 P, length, vocab]`` and ``tokens`` ``[2 P, length]``, or
    packed ``[rows, vocab]`` and ``[rows]`` with ``cu_seqlens`` ``[2 P + 1]``
    (rows outside of it get a zero gradient; offsets that do not rise within
    the rows make the loss NaN).

        s    = sum of a sequence's log-probabilities (mean where length_normalized)
        h    = beta ((s_chosen - ref_chosen) - (s_rejected - ref_rejected))
        loss = mean(-(1 - eps) log sigmoid(h) - eps log sigmoid(-h)),  eps = label_smoothing

    ``ref_logp`` ``[2 P]`` holds the reference model's s; without it, zeros."""
    what, dev = "preference_loss", logits.device
    _check_logits(what, logits)
    if cu_seqlens is None:
        if logits.dim() != 3 or logits.shape[0] < 2 or logits.shape[0] % 2:
            raise ValueError(f"preference_loss: logits of shape {tuple(logits.shape)}; expected [2 pairs, length, vocab], "
                             "or [rows, vocab] with cu_seqlens")
        sequences, length = logits.shape[0], logits.shape[1]
    else:
        if logits.dim() != 2:
            raise ValueError(f"preference_loss: packed logits of shape {tuple(logits.shape)}; expected [rows, vocab]")
        if cu_seqlens.dim() != 1 or cu_seqlens.numel() < 3 or cu_seqlens.numel() % 2 == 0:
            raise ValueError(f"preference_loss: cu_seqlens of shape {tuple(cu_seqlens.shape)}; expected [2 pairs + 1]")
        cu_seqlens = _check_ids(what, "cu_seqlens", cu_seqlens, cu_seqlens.shape, dev)
        sequences, length = cu_seqlens.numel() - 1, 0
    tokens = _check_ids(what, "tokens", tokens, logits.shape[:-1], dev)
    ref = _check_rows(what, "ref_logp", ref_logp, (sequences,), dev)
    p = {"pairs": sequences // 2, "length": length, "beta": _check_number(what, "beta", beta, 0.0),
         "label_smoothing": _check_number(what, "label_smoothing", label_smoothing, 0.0, 1.0),
         "length_normalized": bool(length_normalized), "temperature": _check_temperature(what, temperature)}
    if not logits.is_cuda:
        loss, rewards = _cpu_preference_loss(logits, tokens, ref, cu_seqlens, p)
    else:
        if _is_tracing() or forward_ad._current_level >= 0:
            _check_modes(what, logits, ref_logp)
        call = _PairsCall(logits, tokens, ref, cu_seqlens, p)
        loss, rewards = _run(call, logits, _needs_grad(logits)), call.rewards
    return PreferenceLoss(loss, *rewards.split(p["pairs"]))


@traced("distill_loss")
def distill_loss(logits: torch.Tensor, teacher_ids: torch.Tensor, teacher_logits: torch.Tensor, *,
                 weights: torch.Tensor | None = None, temperature: float = 1.0, denom=None) -> DistillLoss:
    """Distillation from a teacher's top entries (up to 1024 a row):

        q    = softmax(teacher_logits / temperature) over the row's entries
        kl   = sum_k q_k (log q_k - log softmax(logits / temperature)[id_k])
        loss = sum(weights kl) / denom

    ``teacher_ids`` and ``teacher_logits`` (logits or log-probabilities, bf16,
    fp16 or fp32) are ``[..., K]``; a negative id is padding. An id that stands
    in a row twice counts with both shares. A row without entries has loss and
    gradient zero. ``weights`` and ``denom`` as in :func:`policy_loss`; without
    ``denom``, the sum of the weights of all rows."""
    what, dev = "distill_loss", logits.device
    _check_logits(what, logits)
    if teacher_ids.dim() < 1 or not 1 <= teacher_ids.shape[-1] <= MAX_TOP:
        raise ValueError(f"distill_loss: teacher_ids of shape {tuple(teacher_ids.shape)}; expected 1 to {MAX_TOP} entries a row")
    shape = logits.shape[:-1]
    ids = _check_ids(what, "teacher_ids", teacher_ids, (*shape, teacher_ids.shape[-1]), dev)
    if teacher_logits.dtype not in _DTYPES:
        raise TypeError(f"distill_loss: teacher_logits are {teacher_logits.dtype}; expected bfloat16, float16 or float32")
    if teacher_logits.shape != ids.shape or teacher_logits.device != dev:
        raise ValueError(f"distill_loss: teacher_logits {tuple(teacher_logits.shape)} on {teacher_logits.device} do not "
                         f"match teacher_ids {tuple(ids.shape)} on {dev}")
    if teacher_logits.requires_grad:
        raise ValueError("distill_loss: teacher_logits require a gradient, and this loss gives none to them; detach them")
    teacher = teacher_logits.contiguous()
    weights = _check_rows(what, "weights", weights, shape, dev, any_type=True)
    p = {"temperature": _check_temperature(what, temperature), "denom": _check_denom(what, denom, dev)}
    if not logits.is_cuda:
        return DistillLoss(*_cpu_distill_loss(logits, ids, teacher, weights, p))
    if _is_tracing() or forward_ad._current_level >= 0:
        _check_modes(what, logits, teacher_logits, weights, denom)
    needs_grad = _needs_grad(logits)
    kl = torch.empty(shape, dtype=torch.float32, device=dev)
    call = _Call(DISTILL, logits, ids, p["temperature"], kl.new_empty(()), None, kl, None, (None, None, None, weights), teacher,
                 p["denom"], fused=needs_grad)
    return DistillLoss(_run(call, logits, needs_grad), kl)
