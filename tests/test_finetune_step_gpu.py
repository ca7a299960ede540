"""The operators around the two hot paths together, as a trainer runs them: a small model's trunk with a trained table, the vocabulary
loss, an objective, the backward pass and the optimizer's step; against the same model in plain torch (stock eager attention, logits,
elementary operations), fp32.  The attention and the vocabulary loss bound what may differ: 1e-3 of the largest gradient and 1e-4 of a
loss, as in tests/test_wrapper_adapter.py."""
import copy
import subprocess
import sys
from pathlib import Path

import pytest
import torch

from mlx_train_perf_b200 import AdamW, AdapterError, enable_flash_attention
from mlx_train_perf_b200.adapters import torch_lm
from mlx_train_perf_b200.adapters.torch_lm import make_loss_fn, make_policy_loss_fn, make_preference_loss_fn, make_token_loss_fn
from mlx_train_perf_b200.core.loss import VJP_CALLS, check_device_status

transformers = pytest.importorskip("transformers")

VOCAB = 512


def _pair(dev, **over):
    """(stock, ours): the same random model twice, ours with the package's attention."""
    kw = dict(vocab_size=VOCAB, hidden_size=256, intermediate_size=512, num_hidden_layers=2, num_attention_heads=4,
              num_key_value_heads=2, max_position_embeddings=512, attention_dropout=0.0)
    kw.update(over)
    torch.manual_seed(0)
    stock = transformers.LlamaForCausalLM(transformers.LlamaConfig(**kw)).to(dev).float()
    stock.config._attn_implementation = "eager"
    ours = copy.deepcopy(stock)
    enable_flash_attention(ours)
    return stock, ours


def _batch(dev, rows=4, length=70):
    g = torch.Generator().manual_seed(1)
    batch = torch.randint(1, VOCAB, (rows, length + 1), generator=g).to(dev)
    first = torch.randint(1, 20, (rows, 1), generator=g)
    last = torch.randint(30, length + 1, (rows, 1), generator=g)
    return batch, torch.cat([first, last], dim=1).to(dev)


def _plain_logps(model, batch, lengths):
    logits = model(batch[:, :-1]).logits.float()
    steps = torch.arange(1, batch.shape[1], device=batch.device)
    mask = (steps >= lengths[:, 0:1]) & (steps <= lengths[:, 1:2])
    return logits.log_softmax(-1).gather(-1, batch[:, 1:, None])[..., 0], mask


def _gradients_agree(ours, stock):
    for (name, p), (_, q) in zip(ours.named_parameters(), stock.named_parameters()):
        assert (p.grad is None) == (q.grad is None), name
        if p.grad is not None:
            assert (p.grad - q.grad).abs().max() <= 1e-3 * q.grad.abs().max() + 1e-7, name


@pytest.mark.gpu
@pytest.mark.parametrize("tied", [False, True])
def test_preference_and_policy_steps(cuda_device, tied):
    dev = cuda_device
    stock, ours = _pair(dev, tie_word_embeddings=tied)
    batch, lengths = _batch(dev)
    with torch.no_grad():
        ref, old = (x + 0.1 * torch.randn(x.shape, generator=torch.Generator(device=dev).manual_seed(k), device=dev)
                    for k in (1, 2) for x in [make_token_loss_fn(ours)(ours, batch, lengths)[0]])
    a = torch.tensor([[1.0], [-0.5], [0.3], [-2.0]], device=dev)
    calls = dict(VJP_CALLS)
    for which in ("preference", "policy"):
        ours.zero_grad(), stock.zero_grad()
        x, mask = _plain_logps(stock, batch, lengths)
        w = mask.float()
        if which == "preference":
            got = make_preference_loss_fn(ours, beta=0.3, average=True)(ours, batch, lengths, ref).loss
            l = ((x + ref) * w).sum(1) / w.sum(1)
            want = -torch.nn.functional.logsigmoid(0.3 * (l[:2] - l[2:])).mean()
        else:
            got = make_policy_loss_fn(ours, kl_coef=0.2, normalize="sequence")(ours, batch, lengths, old, a, ref).loss
            ratio, z = (x + old).exp(), -ref - x
            f = -torch.minimum(ratio * a, ratio.clamp(0.8, 1.2) * a) + 0.2 * (torch.expm1(z) - z)
            want = ((f * w).sum(1) / w.sum(1)).mean()
        got.backward()
        want.backward()
        assert abs(got.item() - want.item()) < 1e-4 * max(1.0, abs(want.item()))
        _gradients_agree(ours, stock)
    check_device_status()
    for key in ("preference_loss", "policy_loss"):
        assert VJP_CALLS[key] == calls.get(key, 0) + 1
    assert VJP_CALLS["embedding_lookup"] == calls.get("embedding_lookup", 0) + 2


@pytest.mark.gpu
def test_steps_of_a_full_fine_tune(cuda_device):
    """Three steps with AdamW beside torch's on the stock model.  Adam divides a gradient by its own size, so weights move by about lr a
    step whatever the gradient; where a gradient is all rounding its sign is too: twice 3 lr bounds any weight, and the
    mean is held to a hundredth of that."""
    dev = cuda_device
    stock, ours = _pair(dev)
    batch, lengths = _batch(dev)
    theirs, opt = torch.optim.AdamW(stock.parameters(), lr=1e-3), AdamW(ours.parameters(), lr=1e-3)
    for _ in range(3):
        opt.zero_grad(), theirs.zero_grad()
        make_loss_fn(ours)(ours, batch, lengths)[0].backward()
        x, mask = _plain_logps(stock, batch, lengths)
        (-(x * mask).sum() / mask.sum()).backward()
        opt.step(), theirs.step()
    for p, q in zip(ours.parameters(), stock.parameters()):
        off = (p - q).abs()
        assert off.max() <= 6.5e-3 and off.mean() <= 6e-5


@pytest.mark.gpu
def test_8_bit_step_runs_in_bf16(cuda_device):
    dev = cuda_device
    _, ours = _pair(dev)
    ours = ours.to(torch.bfloat16)
    batch, lengths = _batch(dev)
    opt = AdamW(ours.parameters(), lr=1e-3, bits=8, master=True)
    before = [p.detach().clone() for p in ours.parameters()]
    for _ in range(2):
        opt.zero_grad()
        loss, _ = make_loss_fn(ours)(ours, batch, lengths)
        loss.backward()
        norm = torch.nn.utils.get_total_norm([p.grad for p in ours.parameters()])
        opt.step(grad_scale=(1.0 / norm.float().clamp(min=1.0)).reshape(1))
    check_device_status()
    assert all(torch.isfinite(p).all() for p in ours.parameters())
    assert all(not torch.equal(p, b) for p, b in zip(ours.parameters(), before))


@pytest.mark.gpu
def test_which_tables_the_walk_looks_up(cuda_device):
    """Frozen, hooked, norm-limited or wrapped tables stay with their module."""
    mod = torch.nn.Embedding(10, 8).to(cuda_device)
    assert torch_lm._trains_plain_table(mod)
    with torch.no_grad():
        assert not torch_lm._trains_plain_table(mod)
    hook = mod.register_forward_hook(lambda *a: None)
    assert not torch_lm._trains_plain_table(mod)
    hook.remove()
    hook = torch.nn.modules.module.register_module_forward_hook(lambda *a: None)
    assert not torch_lm._trains_plain_table(mod)
    hook.remove()
    assert torch_lm._trains_plain_table(mod)
    for other in (torch.nn.Embedding(10, 8, max_norm=1.0), torch.nn.Embedding(10, 8, sparse=True), torch.nn.Embedding(10, 8, scale_grad_by_freq=True),
                  torch.nn.Embedding(10, 8).half(), torch.nn.Sequential(mod), torch.nn.Embedding(10, 8).requires_grad_(False)):
        assert not torch_lm._trains_plain_table(other.to(cuda_device))
    assert not torch_lm._trains_plain_table(torch.nn.Embedding(10, 8))

    class Sharded(torch.Tensor):
        pass

    mod.weight = torch.nn.Parameter(torch.zeros(10, 8, device=cuda_device).as_subclass(Sharded))
    assert isinstance(mod.weight, Sharded) and not torch_lm._trains_plain_table(mod)


def test_the_walk_s_rows_are_the_module_s_own(monkeypatch):
    """Its check of the ids among them: with a table that the walk trains, an id outside the vocabulary still stops the program."""
    inner = torch.nn.Module()
    inner.embed_tokens, inner.layers, inner.norm = torch.nn.Embedding(10, 4, padding_idx=2), torch.nn.ModuleList(), torch.nn.Identity()
    monkeypatch.setattr(torch_lm, "_trains_plain_table", lambda mod: True)
    ids = torch.tensor([[1, 2, 9], [0, 0, 3]])
    rows = torch_lm._walk(inner, ids, None)
    assert torch.equal(rows, inner.embed_tokens(ids)) and rows.requires_grad
    for bad in (10, -1):
        with pytest.raises(IndexError):
            torch_lm._walk(inner, torch.tensor([[1, bad]]), None)


def test_a_class_s_forward_replaced_before_the_import():
    """Even by a function that carries the old one's name."""
    code = """
import functools, torch
own = torch.nn.Embedding.forward
if {replace}:
    torch.nn.Embedding.forward = functools.wraps(own)(lambda self, ids: 3.0 * own(self, ids))
from mlx_train_perf_b200.adapters import torch_lm
print(torch_lm._has_own_forward(torch.nn.Embedding(3, 2)))
"""
    for replace in (True, False):
        got = subprocess.run([sys.executable, "-c", code.format(replace=replace)], capture_output=True, text=True, check=True,
                             cwd=Path(torch_lm.__file__).parents[2])
        assert got.stdout.strip() == str(not replace)


@pytest.mark.gpu
@pytest.mark.parametrize("padding", [None, 3, 9, -1, -10])
def test_the_walk_s_table_gradient(cuda_device, padding):
    """The module's own rows with the package's gradient, a padding id given from either end; whole numbers, so that sums are exact."""
    inner = torch.nn.Module()
    inner.embed_tokens, inner.layers, inner.norm = torch.nn.Embedding(10, 8).to(cuda_device), torch.nn.ModuleList(), torch.nn.Identity()
    table = inner.embed_tokens
    table.padding_idx = padding
    for rows in (2, 40):
        ids = torch.randint(0, 10, (rows, 5), generator=torch.Generator().manual_seed(rows)).to(cuda_device)
        dy = torch.randint(-4, 5, (rows, 5, 8), generator=torch.Generator().manual_seed(3)).float().to(cuda_device)
        calls = VJP_CALLS.get("embedding_lookup", 0)
        out = torch_lm._walk(inner, ids, None)
        got, = torch.autograd.grad(out, table.weight, dy)
        want, = torch.autograd.grad(torch.nn.functional.embedding(ids, table.weight, padding_idx=padding), table.weight, dy)
        assert torch.equal(out, table(ids)) and torch.equal(got, want) and VJP_CALLS["embedding_lookup"] == calls + 1


@pytest.mark.gpu
@pytest.mark.parametrize("where", ["instance", "class"])
def test_a_forward_put_in_place_of_the_table_s_own(cuda_device, monkeypatch, where):
    """As tools that wrap modules in place do it: the walk's rows are that function's, and so is the table's gradient."""
    dev = cuda_device
    stock, ours = _pair(dev)
    batch, lengths = _batch(dev)
    own = torch.nn.Embedding.forward
    if where == "class":
        monkeypatch.setattr(torch.nn.Embedding, "forward", lambda self, ids: 3.0 * own(self, ids) + 0.01)
    else:
        for model in (stock, ours):
            table = model.model.embed_tokens
            table.forward = lambda ids, table=table: 3.0 * own(table, ids) + 0.01
    assert not torch_lm._trains_plain_table(ours.model.embed_tokens)
    got, _ = make_loss_fn(ours)(ours, batch, lengths)
    x, mask = _plain_logps(stock, batch, lengths)
    want = -(x * mask).sum() / mask.sum()
    got.backward()
    want.backward()
    assert abs(got.item() - want.item()) < 1e-4 * max(1.0, abs(want.item()))
    _gradients_agree(ours, stock)


@pytest.mark.gpu
def test_planner_measures_with_the_package_optimizer(cuda_device):
    """One small point of the planner's measuring command, moments of either width: 8 bits take less, and both run."""
    from mlx_train_perf_b200.plan import estimate as E
    from mlx_train_perf_b200.plan.measure import measure_point
    kw = dict(vocab_size=2000, hidden_size=512, intermediate_size=512, num_hidden_layers=2, num_attention_heads=8, num_key_value_heads=2,
              max_position_embeddings=512, attention_dropout=0.0, tie_word_embeddings=False)
    shape = E.ModelShape.from_config(kw)
    cfg = lambda bits: E.TrainConfig(batch=1, seq_len=256, dtype="bfloat16", lora_rank=64, lora_layers=2, grad_checkpoint=False,
                                     impl="kernel", attention="flash", optimizer_bits=bits)
    peaks = [measure_point(kw, shape, cfg(bits), cuda_device) for bits in (32, 8)]
    assert 0 < peaks[1] <= peaks[0]


def test_planner_books_the_moments_of_either_width():
    from mlx_train_perf_b200.errors import PlanInputError
    from mlx_train_perf_b200.plan import estimate as E
    from mlx_train_perf_b200.plan.calibration import load_calibration
    calib = load_calibration()
    shape = E.ModelShape(vocab=32000, hidden=2048, layers=8, intermediate=5632, heads=16, kv_heads=4, tied=False, quant_bits=None, quant_group=None)
    cfg = lambda bits: E.TrainConfig(batch=1, seq_len=2048, dtype="bfloat16", lora_rank=8, lora_layers=8, grad_checkpoint=True, impl="kernel",
                                     attention="flash", optimizer_bits=bits)
    params = 8 * 2 * 2 * 8 * 2048
    assert E.estimate_peak(shape, cfg(32), calib)[1]["optimizer"] == 8 * params
    assert E.estimate_peak(shape, cfg(8), calib)[1]["optimizer"] == params * 2 + params * 8 // 256
    with pytest.raises(PlanInputError, match="optimizer_bits"):
        E.estimate_peak(shape, cfg(16), calib)


def test_objective_functions_want_a_wrapped_model():
    torch.manual_seed(0)
    m = transformers.LlamaForCausalLM(transformers.LlamaConfig(vocab_size=64, hidden_size=128, intermediate_size=128, num_hidden_layers=1,
                                                               num_attention_heads=2, num_key_value_heads=1, attention_dropout=0.0))
    for make in (make_token_loss_fn, make_preference_loss_fn, make_policy_loss_fn):
        with pytest.raises(AdapterError, match="enable_flash_attention"):
            make(m)
