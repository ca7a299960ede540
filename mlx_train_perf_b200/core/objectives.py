"""Objectives over per-token log-probabilities: `preference_loss` (pairs of sequences) and `policy_loss` (clipped, with a
KL term), each with its gradient, for trainers that go on from the per-token losses of `fused_linear_ce`.

Both take the tokens of S sequences either as (S, L) rows or packed, as (T,) with `cu_seqlens` (S + 1 rising borders);
sequences may be empty.  `mask` (bool, like the tokens) says which tokens count; one that does not takes no part whatever
it holds and gets a zero gradient, and so do packed tokens outside every sequence.  Only `logps` carries a gradient.
`from_nll=True`: all log-probabilities are given as losses `-log p`, as `fused_linear_ce` returns them, and the gradient
is that of the losses.

The reference trains with the masked mean alone (adapters/mlx_lm.py:192-216); these two are further reductions of the
same per-token values.  Nothing here synchronises with the host unless `validate_seqlens` asks for it.
"""
from __future__ import annotations

import ctypes as C
from functools import partial
from typing import Literal, NamedTuple

import torch

from mlx_train_perf_b200 import _lib
from mlx_train_perf_b200.core.loss import VJP_CALLS, has_tangent
from mlx_train_perf_b200.errors import LossInputError

_PREFERENCES = {"sigmoid": 0, "hinge": 1, "squared": 2}
_KLS = {"k1": 0, "k2": 1, "k3": 2}
_NORMALIZE = {"token": 0, "sequence": 1, "sum": 2}
_DTYPES = (torch.float32, torch.bfloat16)


class PreferenceLoss(NamedTuple):
    """`loss` (scalar, differentiable) and the rewards beta * l of each pair's two sequences, (P,) each, fp32."""
    loss: torch.Tensor
    chosen_rewards: torch.Tensor
    rejected_rewards: torch.Tensor


class PolicyLoss(NamedTuple):
    """`loss` (scalar, differentiable); the mean KL term and the share of clipped tokens over the tokens that count."""
    loss: torch.Tensor
    kl: torch.Tensor
    clip_fraction: torch.Tensor


def _unit_inner(t: torch.Tensor) -> torch.Tensor:
    return t if t.is_contiguous() or t.stride(-1) == 1 or t.shape[-1] <= 1 else t.contiguous()


def _check_tokens(logps: torch.Tensor, cu_seqlens: torch.Tensor | None, validate_seqlens: bool) -> int:
    """The number of sequences."""
    if has_tangent(logps):
        raise LossInputError("this loss has no forward-mode derivative")
    if not logps.is_cuda:
        raise LossInputError(f"logps must be a CUDA tensor (the operators have no CPU path); got {logps.device}")
    if logps.dtype not in _DTYPES:
        raise LossInputError(f"logps must be fp32 or bf16, got {logps.dtype}")
    if cu_seqlens is None:
        if logps.ndim != 2 or logps.shape[0] < 1:
            raise LossInputError(f"logps must be (S, L) with at least one sequence, or (T,) with cu_seqlens; got {tuple(logps.shape)}")
        return logps.shape[0]
    if logps.ndim != 1:
        raise LossInputError(f"with cu_seqlens, logps must be (T,) packed tokens; got {tuple(logps.shape)}")
    if (cu_seqlens.ndim != 1 or cu_seqlens.shape[0] < 2 or cu_seqlens.dtype not in (torch.int32, torch.int64)
            or cu_seqlens.device != logps.device):
        raise LossInputError("cu_seqlens must be (S + 1,) int32 or int64 with S >= 1, on logps' device; got "
                             f"{tuple(cu_seqlens.shape)} {cu_seqlens.dtype} on {cu_seqlens.device}")
    if validate_seqlens:
        cu = cu_seqlens.to(torch.int64)
        if int(cu[0]) < 0 or int(cu[-1]) > logps.shape[0] or bool((cu[1:] < cu[:-1]).any()):
            raise LossInputError(f"cu_seqlens must rise from 0 or more to at most T={logps.shape[0]}")
    return cu_seqlens.shape[0] - 1


def _check_like(name: str, t: torch.Tensor, logps: torch.Tensor) -> torch.Tensor:
    if t.shape != logps.shape or t.device != logps.device:
        raise LossInputError(f"{name} must match logps: {tuple(logps.shape)} on {logps.device}, got {tuple(t.shape)} on {t.device}")
    return _unit_inner(t)


def _check_mask(mask: torch.Tensor | None, logps: torch.Tensor) -> torch.Tensor | None:
    if mask is None:
        return None
    if mask.dtype != torch.bool:
        raise LossInputError(f"mask must be bool, got {mask.dtype}")
    return _check_like("mask", mask, logps)


def _check_other(name: str, t: torch.Tensor | None, logps: torch.Tensor) -> torch.Tensor | None:
    if t is None:
        return None
    if t.dtype not in _DTYPES:
        raise LossInputError(f"{name} must be fp32 or bf16, got {t.dtype}")
    return _check_like(name, t, logps)


def _contiguous(shape, dtype, device) -> torch.Tensor:
    """torch.empty of one or two dimensions; given its strides it is 2 us cheaper."""
    return torch.empty_strided(shape, (1,) if len(shape) == 1 else (shape[1], 1), dtype=dtype, device=device)


def _row_stride(t: torch.Tensor | None) -> int:
    return 0 if t is None or t.ndim == 1 else t.stride(0)


class _Call:
    """What one call hands the library, and what it got back.  The autograd functions below take it as their one argument beside
    `logps`: every further argument and output costs a training step host time (12 arguments and 3 outputs: 15 us of it)."""
    __slots__ = ("seqs", "mask", "cu", "old", "ref", "adv", "adv_strides", "rule", "from_nll", "per_sequence", "recorded", "out",
                 "at", "slopes_at", "shape", "dtype", "slopes")

    def args(self, logps) -> _lib.ObjectiveArgs:
        mask, cu, old, ref, adv = self.mask, self.cu, self.old, self.ref, self.adv
        other = ref if old is None else old
        return _lib.ObjectiveArgs(
            logps.data_ptr(), None if old is None else old.data_ptr(), None if ref is None else ref.data_ptr(),
            None if mask is None else mask.data_ptr(), None if adv is None else adv.data_ptr(),
            None if cu is None else cu.data_ptr(), self.seqs, logps.shape[-1], _row_stride(logps), _row_stride(old),
            _row_stride(ref), _row_stride(mask), *self.adv_strides, logps.dtype == torch.bfloat16,
            other is not None and other.dtype == torch.bfloat16, cu is not None and cu.dtype == torch.int64, self.from_nll)

    def buffer(self, lib, a, logps, slopes: bool) -> tuple[torch.Tensor, int, int, int]:
        """One allocation for the workspace, the weights of sequences or of the batch, and the tokens' slopes: (buffer, workspace bytes,
        address of the weights, address of the slopes or 0)."""
        with _lib.on(logps.device):                       # the blocks go by that device's SMs
            nbytes = lib.b200tp_objective_workspace_bytes(C.byref(a))
        self.at = nbytes // 4
        self.slopes_at = self.at + ((self.seqs if self.per_sequence else 1) + 3) // 4 * 4     # on a boundary of 16 bytes
        size = self.slopes_at + (logps.numel() if slopes else 0)
        buf = torch.empty_strided((size,), (1,), dtype=torch.float32, device=logps.device)
        base = buf.data_ptr()
        return buf, nbytes, base + nbytes, base + 4 * self.slopes_at if slopes else 0

    def keep(self, ctx, logps, buf, slopes: bool):
        """Everything the gradient needs, apart from what the caller is given and may write to; the inputs are let go."""
        ctx.save_for_backward(buf, self.mask, self.cu)
        ctx.call, self.shape, self.dtype, self.slopes = self, logps.shape, logps.dtype, slopes
        self.mask = self.cu = self.old = self.ref = self.adv = None

    def gradient(self, ctx, g):
        """Gradient for logps from the loss's upstream gradient.  Addresses are those of the tensors that autograd hands back."""
        if torch.is_grad_enabled():
            raise LossInputError("this loss has no second derivative (create_graph=True)")
        buf, mask, cu = ctx.saved_tensors
        dev, dtype = buf.device, self.dtype
        grad = _contiguous(self.shape, dtype, dev)
        at = grad.data_ptr()                              # logps is not read any more
        a = _lib.ObjectiveArgs(at, None, None, None if mask is None else mask.data_ptr(), None, None if cu is None else cu.data_ptr(),
                               self.seqs, self.shape[-1], 0, 0, 0, _row_stride(mask), 0, 0, dtype is torch.bfloat16, 0,
                               cu is not None and cu.dtype is torch.int64, 0)
        if g.dtype is not torch.float32:
            g = g.to(torch.float32)
        base = buf.data_ptr()
        weights, slopes = base + 4 * self.at, base + 4 * self.slopes_at if self.slopes else None
        with _lib.on(dev):
            rc = _lib.load().b200tp_objective_bwd(C.byref(a), slopes, weights, self.per_sequence, g.data_ptr(), at, _lib.stream(dev))
        _lib.check(rc)
        return grad


class _Preference(torch.autograd.Function):
    """logps -> loss; `call.out` gets the rewards.  Keeps a weight for each sequence.  Without a gradient `forward` is called by
    itself (`ctx` None)."""

    @staticmethod
    def forward(ctx, logps, call):
        lib = _lib.load()
        dev = logps.device
        a = call.args(logps)
        loss = torch.empty_strided((), (), dtype=torch.float32, device=dev)
        call.out = torch.empty_strided((call.seqs,), (1,), dtype=torch.float32, device=dev)
        buf, nbytes, weights, _ = call.buffer(lib, a, logps, False)
        with _lib.on(dev):
            rc = lib.b200tp_preference_loss_fwd(C.byref(a), *call.rule, loss.data_ptr(), call.out.data_ptr(), weights, buf.data_ptr(),
                                                nbytes, _lib.stream(dev))
        _lib.check(rc)
        if call.recorded:
            call.keep(ctx, logps, buf, False)
        return loss

    @staticmethod
    def backward(ctx, g):
        VJP_CALLS["preference_loss"] = VJP_CALLS.get("preference_loss", 0) + 1
        return ctx.call.gradient(ctx, g), None


class _Policy(torch.autograd.Function):
    """logps -> loss; `call.out` gets the mean KL term and the clipped share.  Keeps a slope for each token, where a gradient may be
    asked for."""

    @staticmethod
    def forward(ctx, logps, call):
        lib = _lib.load()
        dev = logps.device
        a = call.args(logps)
        loss = torch.empty_strided((), (), dtype=torch.float32, device=dev)
        stats = torch.empty_strided((2,), (1,), dtype=torch.float32, device=dev)
        buf, nbytes, weights, slopes = call.buffer(lib, a, logps, call.recorded)
        with _lib.on(dev):
            rc = lib.b200tp_policy_loss_fwd(C.byref(a), *call.rule, loss.data_ptr(), stats.data_ptr(), slopes or None, weights,
                                            buf.data_ptr(), nbytes, _lib.stream(dev))
        _lib.check(rc)
        call.out = stats[0], stats[1]
        if call.recorded:
            call.keep(ctx, logps, buf, True)
        return loss

    @staticmethod
    def backward(ctx, g):
        VJP_CALLS["policy_loss"] = VJP_CALLS.get("policy_loss", 0) + 1
        return ctx.call.gradient(ctx, g), None


def _call(logps, seqs, mask, cu_seqlens, old, ref, rule, from_nll, per_sequence) -> _Call:
    call = _Call()
    call.seqs, call.mask, call.cu = seqs, mask, None if cu_seqlens is None else cu_seqlens.contiguous()
    call.old, call.ref = old, ref
    call.adv, call.adv_strides, call.rule, call.from_nll, call.per_sequence = None, (0, 0), rule, bool(from_nll), per_sequence
    call.recorded = torch.is_grad_enabled() and logps.requires_grad
    return call


def preference_loss(logps: torch.Tensor, ref_logps: torch.Tensor | None = None, *, mask: torch.Tensor | None = None,
                    cu_seqlens: torch.Tensor | None = None, kind: Literal["sigmoid", "hinge", "squared"] = "sigmoid",
                    beta: float = 0.1, label_smoothing: float = 0.0, margin: float = 0.0, average: bool = False,
                    from_nll: bool = False, validate_seqlens: bool = False) -> PreferenceLoss:
    """Mean loss over P pairs; sequence i is preferred to sequence P + i (S = 2 P: first the chosen, then the rejected).

    With l_s the sum over the sequence's tokens of `logps - ref_logps` (`average`: its mean; no `ref_logps`: of
    `logps`) and h = beta (l_i - l_{P+i}) - margin:
      sigmoid  (1 - e) log(1 + exp(-h)) + e log(1 + exp(h)), e = `label_smoothing`
      hinge    max(0, 1 - h)
      squared  ((h - 1/2) / beta)^2
    A sequence without a token that counts has l = 0.  `cu_seqlens` is trusted (borders outside [0, T] are held there, ones that do
    not rise leave the gradient of tokens between them undefined); `validate_seqlens=True` checks it, with a host synchronisation."""
    seqs = _check_tokens(logps, cu_seqlens, validate_seqlens)
    if seqs % 2 != 0:
        raise LossInputError(f"a preference loss needs pairs: an even number of sequences, got {seqs}")
    if kind not in _PREFERENCES:
        raise LossInputError(f"unknown kind {kind!r}; expected one of {sorted(_PREFERENCES)}")
    if not beta > 0.0:
        raise LossInputError(f"beta must be positive, got {beta}")
    if not 0.0 <= label_smoothing < 1.0 or (label_smoothing and kind != "sigmoid"):
        raise LossInputError(f"label_smoothing must lie in [0, 1) and needs kind='sigmoid'; got {label_smoothing} with {kind!r}")
    mask, ref = _check_mask(mask, logps), _check_other("ref_logps", ref_logps, logps)
    rule = (_PREFERENCES[kind], float(beta), float(label_smoothing), float(margin), bool(average))
    call = _call(logps, seqs, mask, cu_seqlens, None, ref, rule, from_nll, True)
    loss = (_Preference.apply if call.recorded else partial(_Preference.forward, None))(_unit_inner(logps), call)
    return PreferenceLoss(loss, call.out[:seqs // 2], call.out[seqs // 2:])


def policy_loss(logps: torch.Tensor, old_logps: torch.Tensor, advantages: torch.Tensor, *,
                ref_logps: torch.Tensor | None = None, mask: torch.Tensor | None = None,
                cu_seqlens: torch.Tensor | None = None, clip_low: float = 0.2, clip_high: float = 0.2,
                kl_coef: float = 0.0, kl: Literal["k1", "k2", "k3"] = "k3",
                normalize: Literal["token", "sequence", "sum"] = "token", from_nll: bool = False,
                validate_seqlens: bool = False) -> PolicyLoss:
    """Per token -min(r A, clip(r, 1 - clip_low, 1 + clip_high) A) + kl_coef * KL with r = exp(logps - old_logps).

    `advantages`: like `logps`, or (S, 1), one for each sequence.  KL of `logps` against `ref_logps`, d their difference:
    k1 d, k2 d^2 / 2, k3 exp(-d) - 1 + d; it is reported also where kl_coef is 0, and 0 without `ref_logps`.
    `normalize`: "token" averages over all tokens that count, "sequence" over each sequence's and then over the S sequences (an
    empty one adds 0), "sum" adds up.  A token is clipped where the clipped term is the smaller one; the comparison is made on
    logps - old_logps against log(1 + clip_high) and log(1 - clip_low).  `cu_seqlens` is trusted as in `preference_loss`."""
    seqs = _check_tokens(logps, cu_seqlens, validate_seqlens)
    if kl not in _KLS:
        raise LossInputError(f"unknown kl {kl!r}; expected one of {sorted(_KLS)}")
    if normalize not in _NORMALIZE:
        raise LossInputError(f"unknown normalize {normalize!r}; expected one of {sorted(_NORMALIZE)}")
    if not (0.0 <= clip_low <= 1.0 and clip_high >= 0.0):
        raise LossInputError(f"clip_low must lie in [0, 1] and clip_high be at least 0; got {clip_low}, {clip_high}")
    if kl_coef != 0.0 and ref_logps is None:
        raise LossInputError("a KL term (kl_coef != 0) needs ref_logps")
    mask, old, ref = (_check_mask(mask, logps), _check_other("old_logps", old_logps, logps),
                      _check_other("ref_logps", ref_logps, logps))
    if ref is not None and ref.dtype is not old.dtype:   # the kernel reads both in one dtype
        old, ref = old.to(torch.float32), ref.to(torch.float32)
    adv = advantages
    if adv.dtype not in _DTYPES or adv.device != logps.device or (adv.shape != logps.shape and tuple(adv.shape) != (seqs, 1)):
        raise LossInputError(f"advantages must be fp32 / bf16, on logps' device and like logps {tuple(logps.shape)} or ({seqs}, 1); "
                             f"got {tuple(adv.shape)} {adv.dtype} on {adv.device}")
    if adv.dtype is not torch.float32:
        adv = adv.to(torch.float32)
    if cu_seqlens is None:
        strides = adv.stride(0), adv.stride(1) if adv.shape[1] == logps.shape[1] else 0
    else:
        strides = (0, adv.stride(0)) if adv.ndim == 1 else (adv.stride(0), 0)
    rule = (float(clip_low), float(clip_high), float(kl_coef), _KLS[kl], _NORMALIZE[normalize])
    call = _call(logps, seqs, mask, cu_seqlens, old, ref, rule, from_nll, normalize == "sequence")
    call.adv, call.adv_strides = adv, strides
    loss = (_Policy.apply if call.recorded else partial(_Policy.forward, None))(_unit_inner(logps), call)
    return PolicyLoss(loss, *call.out)
