"""Trainer loss shims for PyTorch (Hugging-Face style) Llama / Qwen2 / Qwen3 models: the
direct callers of the two operators (src/mlx_train_perf/adapters/mlx_lm.py:140-164
`split_model`, :167-216 `make_loss_fn`, :221-295 `make_packed_loss_fn`).

Both loss functions walk the inner model layer by layer --
`embed_tokens -> layers(h, mask) -> norm` -- so the mask each block sees is exactly "causal" or
a `PackedMask` (a top-level `model(input_ids)` call would hand the blocks a tensor mask, which
the flash wrapper refuses), then feed the hidden states to the fused loss with the logits never
materialised.  Masked mean: loss = sum(nll * mask) / ntoks, reduced inside the library.

`make_token_loss_fn` stops before that reduction; `make_preference_loss_fn` and `make_policy_loss_fn` go on from the
per-token losses with the objectives of `core/objectives.py`.  Where the embedding table is trained, its gradient is
`embedding_lookup`'s, which adds the rows of equal ids in a fixed order.
"""
from __future__ import annotations

from typing import Any, Callable

import torch
from torch.nn.modules.module import _has_any_global_hook

from mlx_train_perf_b200.attention.segments import PackedMask
from mlx_train_perf_b200.attention.wrapper import SUPPORTED_FAMILIES, FlashAttentionWrapper
from mlx_train_perf_b200.core.embedding import module_lookup
from mlx_train_perf_b200.core.loss import (IGNORE_INDEX, DenseHead, HeadRef, QuantizedHead, fused_linear_ce,
                                           reduced_linear_cross_entropy, resolve_impl, tied_head)
from mlx_train_perf_b200.core.objectives import PolicyLoss, PreferenceLoss, policy_loss, preference_loss
from mlx_train_perf_b200.errors import AdapterError


def _head_from_module(mod: Any) -> HeadRef:
    """A `nn.Linear`-like lm_head -> DenseHead; a module carrying the 4-bit affine layout
    (`w_q` / `scales` / `biases` [, `group_size`, `bits`]) -> QuantizedHead."""
    if all(hasattr(mod, a) for a in ("w_q", "scales", "biases")):
        return QuantizedHead(w_q=mod.w_q, scales=mod.scales, biases=mod.biases,
                             group_size=int(getattr(mod, "group_size", 64)), bits=int(getattr(mod, "bits", 4)))
    w = getattr(mod, "weight", None)
    if isinstance(w, torch.Tensor) and w.ndim == 2:
        if getattr(mod, "bias", None) is not None:
            raise AdapterError("lm_head with a bias is not supported by the fused loss")
        return DenseHead(weight=w, trainable=bool(w.requires_grad))
    raise AdapterError(f"unsupported lm_head module type {type(mod).__name__!r}")


def split_model(model: Any) -> tuple[Callable[[torch.Tensor], torch.Tensor], HeadRef]:
    """(hidden-state trunk, HeadRef) of a causal-LM model; `AdapterError` for other shapes."""
    family = getattr(getattr(model, "config", None), "model_type", None)
    if family not in SUPPORTED_FAMILIES:
        raise AdapterError(f"unsupported model architecture (model_type {family!r}); supported: "
                           + ", ".join(SUPPORTED_FAMILIES))
    inner = getattr(model, "model", None)
    if inner is None or not all(hasattr(inner, a) for a in ("embed_tokens", "layers", "norm")):
        raise AdapterError("model.model must expose embed_tokens / layers / norm")
    if getattr(model.config, "tie_word_embeddings", False):
        w = inner.embed_tokens.weight
        head: HeadRef = tied_head(w, trainable=bool(w.requires_grad))
    else:
        head = _head_from_module(model.lm_head)

    def trunk(input_ids: torch.Tensor) -> torch.Tensor:
        return _walk(inner, input_ids, "causal")

    return trunk, head


def _has_own_forward(mod: torch.nn.Embedding) -> bool:
    """Whether calling `mod` runs torch's own code: no `forward` on the instance, and none put in the class's place at any time, this
    module's import included."""
    code = getattr(torch.nn.Embedding.forward, "__code__", None)
    return "forward" not in vars(mod) and code is not None and code.co_filename == torch.nn.modules.sparse.__file__


def _trains_plain_table(mod: Any) -> bool:
    """Whether `embed_tokens` is a plain nn.Embedding with a trained fp32 / bf16 table on a GPU and nothing attached to it: then
    `embedding_lookup` gives the same gradient (summed in fp32 in a fixed order, rounded once).  Anything
    else (frozen, wrapped by an adapter, hooked, with a `forward` put in place of its own, sharded, norm-limited, sparse) stays the
    module's own."""
    if type(mod) is not torch.nn.Embedding or not torch.is_grad_enabled() or _has_any_global_hook():
        return False
    if not _has_own_forward(mod):
        return False
    w = mod.weight
    return (type(w) in (torch.Tensor, torch.nn.Parameter) and w.is_cuda and w.requires_grad and w.dtype in (torch.float32, torch.bfloat16)
            and mod.max_norm is None and not mod.sparse and not mod.scale_grad_by_freq
            and not torch.is_autocast_enabled("cuda")
            and not (mod._forward_hooks or mod._forward_pre_hooks or mod._backward_hooks or mod._backward_pre_hooks))


def _walk(inner: Any, input_ids: torch.Tensor, mask: Any) -> torch.Tensor:
    table = inner.embed_tokens
    if _trains_plain_table(table):
        h = module_lookup(table, input_ids)
    else:
        h = table(input_ids)
    b, length = input_ids.shape
    pos = torch.arange(length, device=input_ids.device)[None].expand(b, -1)   # never reset per segment
    rope = inner.rotary_emb(h, pos) if hasattr(inner, "rotary_emb") else None
    for layer in inner.layers:
        out = layer(h, attention_mask=mask, position_ids=pos, position_embeddings=rope)
        h = out[0] if isinstance(out, tuple) else out
    return inner.norm(h)


def _require_wrapped(model: Any, who: str) -> None:
    for i, layer in enumerate(model.model.layers):
        if not isinstance(layer.self_attn, FlashAttentionWrapper):
            raise AdapterError(f"{who} requires enable_flash_attention(model) first; layer {i} self_attn is "
                               f"{type(layer.self_attn).__name__!r}")


def _supervised(batch: torch.Tensor, lengths: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """(mask, targets) of a (B, L+1) batch: position s (1-based, on the target axis) counts iff offset <= s <= length; the others'
    targets are the ignored index."""
    targets = batch[:, 1:]
    steps = torch.arange(1, targets.shape[1] + 1, device=targets.device)
    mask = (steps >= lengths[:, 0:1]) & (steps <= lengths[:, 1:2])
    return mask, torch.where(mask, targets.to(torch.int64), torch.full_like(targets, IGNORE_INDEX, dtype=torch.int64))


def make_loss_fn(model: Any, *, impl: str = "auto"):
    """`loss(model, batch, lengths) -> (loss, ntoks)`: batch int (B, L+1); lengths int (B, 2)
    = (offset, length) per row; position s (1-based, on the target axis) is supervised iff
    offset <= s <= length."""
    split_model(model)
    _require_wrapped(model, "make_loss_fn")

    def loss_fn(model_arg: Any, batch: torch.Tensor, lengths: torch.Tensor):
        trunk, head = split_model(model_arg)
        hidden = trunk(batch[:, :-1])
        resolve_impl(head=head, dtype=hidden.dtype, n=hidden.shape[0] * hidden.shape[1], d=hidden.shape[-1],
                     impl=impl)
        _, masked_targets = _supervised(batch, lengths)
        # the masked mean (and the token count) are formed inside the library: unsupervised positions carry
        # ignore_index, so loss = sum(nll over supervised positions) / ntoks
        loss, count = reduced_linear_cross_entropy(hidden, head, masked_targets, impl=impl, reduction="mean")
        return loss, count.to(torch.int64)

    return loss_fn


def make_token_loss_fn(model: Any, *, impl: str = "auto"):
    """`loss(model, batch, lengths) -> (nll, mask)`, (B, L) each: the per-token losses -log p of the targets and which positions are
    supervised (the others' are 0); batch and lengths as in `make_loss_fn`.  Under `torch.no_grad()` this is the pass of a reference or
    a sampling model."""
    split_model(model)
    _require_wrapped(model, "make_token_loss_fn")

    def loss_fn(model_arg: Any, batch: torch.Tensor, lengths: torch.Tensor):
        trunk, head = split_model(model_arg)
        hidden = trunk(batch[:, :-1])
        mask, masked_targets = _supervised(batch, lengths)
        return fused_linear_ce(hidden, head, masked_targets, impl=impl)[0], mask

    return loss_fn


def make_preference_loss_fn(model: Any, *, impl: str = "auto", **rule):
    """`loss(model, batch, lengths, ref_nll=None) -> PreferenceLoss`: rows [0, P) of the batch hold the chosen sequences, rows
    [P, 2P) the rejected ones; `ref_nll` (B, L): the reference model's `make_token_loss_fn` losses.  `rule`: the keywords of
    `preference_loss` (kind, beta, label_smoothing, margin, average)."""
    token_losses = make_token_loss_fn(model, impl=impl)

    def loss_fn(model_arg: Any, batch: torch.Tensor, lengths: torch.Tensor, ref_nll: torch.Tensor | None = None) -> PreferenceLoss:
        nll, mask = token_losses(model_arg, batch, lengths)
        return preference_loss(nll, ref_nll, mask=mask, from_nll=True, **rule)

    return loss_fn


def make_policy_loss_fn(model: Any, *, impl: str = "auto", **rule):
    """`loss(model, batch, lengths, old_nll, advantages, ref_nll=None) -> PolicyLoss`: `old_nll`, `ref_nll` (B, L) the sampling and the
    reference model's `make_token_loss_fn` losses, `advantages` (B, L) or (B, 1).  `rule`: the keywords of `policy_loss` (clip_low,
    clip_high, kl_coef, kl, normalize)."""
    token_losses = make_token_loss_fn(model, impl=impl)

    def loss_fn(model_arg: Any, batch: torch.Tensor, lengths: torch.Tensor, old_nll: torch.Tensor, advantages: torch.Tensor,
                ref_nll: torch.Tensor | None = None) -> PolicyLoss:
        nll, mask = token_losses(model_arg, batch, lengths)
        return policy_loss(nll, old_nll, advantages, ref_logps=ref_nll, mask=mask, from_nll=True, **rule)

    return loss_fn


def make_packed_loss_fn(model: Any, *, impl: str = "auto"):
    """`loss(model, batch, seg_id, seg_start, loss_mask) -> (loss, ntoks)` for the 4-tuple
    `packed_iterate_batches` yields; every block gets `PackedMask(seg_id, seg_start)`."""
    split_model(model)
    _require_wrapped(model, "make_packed_loss_fn")

    def loss_fn(model_arg: Any, batch: torch.Tensor, seg_id: torch.Tensor, seg_start: torch.Tensor,
                loss_mask: torch.Tensor):
        _, head = split_model(model_arg)
        inputs, targets = batch[:, :-1], batch[:, 1:]
        hidden = _walk(model_arg.model, inputs, PackedMask(seg_id=seg_id, seg_start=seg_start))
        masked_targets = torch.where(loss_mask, targets.to(torch.int64),
                                     torch.full_like(targets, IGNORE_INDEX, dtype=torch.int64))
        loss, count = reduced_linear_cross_entropy(hidden, head, masked_targets, impl=impl, reduction="mean")
        return loss, count.to(torch.int64)

    return loss_fn
