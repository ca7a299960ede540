"""Refusals of the objectives', the optimizer's and the embedding's C entry points, which come before anything is launched (no GPU needed), and the
Python checks that host tensors reach."""
import ctypes as C

import numpy as np
import pytest
import torch

from mlx_train_perf_b200 import (AdamW, AdamWState, EmbeddingInputError, LossInputError, OptimizerInputError, _lib, embedding_lookup,
                                 policy_loss, preference_loss)
from mlx_train_perf_b200.build import build

PTR = 1 << 20                          # a non-null placeholder: nothing is dereferenced


@pytest.fixture(scope="module")
def lib():
    build(verbose=False)
    return _lib.load()


def _objective(**change):
    a = _lib.ObjectiveArgs(PTR, PTR, PTR, None, PTR, None, 4, 100, 100, 100, 100, 0, 1, 0, 0, 0, 0, 0)
    for k, v in change.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("change,text", [
    ({"seqs": 0}, b"number of sequences"), ({"seqs": 1 << 30}, b"number of sequences"), ({"length": -1}, b"negative length"),
    ({"length": 1 << 40}, b"2^30"), ({"dtype": 7}, b"fp32 or bf16"), ({"other_dtype": 2}, b"fp32 or bf16"), ({"logps": None}, b"logps is null")])
def test_objective_arguments(lib, change, text):
    a = _objective(**change)
    assert lib.b200tp_objective_workspace_bytes(C.byref(a)) == 0
    assert text in lib.b200tp_last_error()
    assert lib.b200tp_preference_loss_fwd(C.byref(a), 0, 0.1, 0.0, 0.0, 0, PTR, PTR, PTR, PTR, 1 << 20, None) == _lib.ERR_LOSS_INPUT
    assert lib.b200tp_policy_loss_fwd(C.byref(a), 0.2, 0.2, 0.0, 2, 0, PTR, PTR, PTR, PTR, PTR, 1 << 20, None) == _lib.ERR_LOSS_INPUT
    assert lib.b200tp_objective_bwd(C.byref(a), None, PTR, 1, PTR, PTR, None) == _lib.ERR_LOSS_INPUT


def test_objective_rules_and_workspace(lib):
    a = _objective()
    need = lib.b200tp_objective_workspace_bytes(C.byref(a))
    assert 0 < need <= 4096 and need % 256 == 0
    pref = lambda a, kind=0, beta=0.1, loss=PTR, ws=PTR, n=need: lib.b200tp_preference_loss_fwd(
        C.byref(a), kind, beta, 0.0, 0.0, 0, loss, PTR, PTR, ws, n, None)
    assert pref(_objective(seqs=3)) == _lib.ERR_LOSS_INPUT and pref(a, kind=3) == _lib.ERR_LOSS_INPUT
    assert pref(a, beta=0.0) == _lib.ERR_LOSS_INPUT and pref(a, beta=float("nan")) == _lib.ERR_LOSS_INPUT and pref(a, loss=None) == _lib.ERR_LOSS_INPUT
    assert pref(a, ws=None) == _lib.ERR_WORKSPACE and pref(a, ws=PTR + 8) == _lib.ERR_WORKSPACE and pref(a, n=need - 1) == _lib.ERR_WORKSPACE
    pol = lambda a, low=0.2, high=0.2, coef=0.1, kl=2, norm=0: lib.b200tp_policy_loss_fwd(
        C.byref(a), low, high, coef, kl, norm, PTR, PTR, PTR, PTR, PTR, need, None)
    for bad in (dict(low=-0.1), dict(low=1.1), dict(high=-1.0), dict(kl=3), dict(norm=3), dict(norm=-1), dict(low=float("nan"))):
        assert pol(a, **bad) == _lib.ERR_LOSS_INPUT, bad
    assert pol(_objective(ref_logps=None)) == _lib.ERR_LOSS_INPUT and b"KL term" in lib.b200tp_last_error()
    assert pol(_objective(old_logps=None)) == _lib.ERR_LOSS_INPUT and pol(_objective(advantages=None)) == _lib.ERR_LOSS_INPUT
    assert lib.b200tp_objective_bwd(C.byref(a), PTR, None, 1, PTR, PTR, None) == _lib.ERR_LOSS_INPUT


def test_workspace_grows_with_sequences_not_tokens(lib):
    """Sums of 32 bytes for each block: at most 512 blocks a sequence and about eight an SM in all."""
    for seqs, length in ((1, 1 << 30), (2, 1 << 20), (512, 8192), (1 << 20, 4)):
        a = _objective(seqs=seqs, length=length)
        assert 32 * seqs <= lib.b200tp_objective_workspace_bytes(C.byref(a)) <= 32 * max(seqs, 2 * 1184) + 256


def _adamw(rows, **change):
    a = _lib.AdamwArgs(PTR, PTR, None, None, PTR, PTR, None, None, 1e-3, 0.9, 0.999, 1e-8, 0.01, 1.0, None, 1, 0, 0, 32, 0)
    for k, v in change.items():
        setattr(a, k, v)
    rows = np.array(rows, dtype=np.int64).reshape(-1, 5)
    return _lib.load().b200tp_adamw_step(C.byref(a), rows.ctypes.data, len(rows), None)


ROW = [PTR, PTR, PTR, 100, 0]


@pytest.mark.parametrize("change", [dict(bits=16), dict(param_dtype=3), dict(grad_dtype=2), dict(step=0), dict(beta1=1.0), dict(beta2=-0.1),
                                    dict(eps=-1.0), dict(lr=-1.0), dict(lr=float("nan")), dict(weight_decay=-0.1), dict(exp_avg=None), dict(exp_avg_sq_out=None),
                                    dict(bits=8), dict(master=PTR), dict(master=PTR, master_out=PTR), dict(exp_avg=PTR + 4), dict(exp_avg_out=PTR + 8)])
def test_adamw_arguments(lib, change):
    assert _adamw([ROW], **change) == _lib.ERR_OPTIM_INPUT


@pytest.mark.parametrize("rows", [
    [[0, PTR, PTR, 100, 0]], [[PTR, 0, PTR, 100, 0]], [[PTR, PTR, 0, 100, 0]], [[PTR, PTR, PTR, -1, 0]], [[PTR, PTR, PTR, 100, 128]],
    [[PTR, PTR, PTR, 100, -256]], [[PTR + 1, PTR, PTR, 100, 0]], [[PTR, PTR + 2, PTR, 100, 0]],
    [ROW, ROW], [ROW, [PTR, PTR, PTR + 396, 100, 256]], [ROW, [PTR, PTR, PTR + 400, 100, 0]], [[PTR, PTR, PTR, 257, 0], [PTR, PTR, PTR + 4096, 8, 256]],
    [[PTR, PTR, PTR + 8, 100, 0]], [[PTR, PTR, PTR + 4096, 100, 0], [PTR + 4196, PTR, PTR + 8192, 100, 256]]])
def test_adamw_tables(lib, rows):
    assert _adamw(rows) == _lib.ERR_OPTIM_INPUT


@pytest.mark.parametrize("rows,change", [
    ([[PTR, PTR + 8, PTR, 100, 0]], {}), ([[PTR, PTR + 4096, PTR, 100, 0], [PTR + 8192, PTR, PTR + 8192, 100, 256]], {}),
    ([[PTR, PTR + 396, PTR, 100, 0]], {}), ([[PTR + 400, PTR + 4, PTR + 400, 100, 0]], {}), ([[PTR, PTR, PTR, 100, 0]], dict(grad_dtype=1)),
    ([[PTR, PTR + 64, PTR + 4096, 100, 0], [PTR + 400, PTR + 4200, PTR + 8192, 100, 256]], {})])
def test_gradients_in_the_way_of_results(lib, rows, change):
    """A gradient that another tensor's results, or its own ones elsewhere, would overwrite while it is read."""
    assert _adamw(rows, **change) == _lib.ERR_OPTIM_INPUT and b"a gradient and a parameter" in lib.b200tp_last_error()


@pytest.mark.parametrize("rows", [
    [[PTR, PTR, PTR, 100, 0]], [[PTR, PTR + 400, PTR, 100, 0]], [[PTR + 400, PTR, PTR + 400, 100, 0]], [[PTR, PTR, PTR + 4096, 100, 0]],
    [[PTR, PTR + 4096, PTR + 4096, 100, 0]], [[PTR, PTR + 4096, PTR, 100, 0], [PTR + 400, PTR + 4096, PTR + 400, 100, 256]]])
def test_gradients_that_are_in_no_way(lib, rows):
    """Beside the results, exactly on them, on read-only parameters, and one gradient for two tensors: the tensors pass, and what is refused
    is the table behind them, whose place in the states is the first one's."""
    assert _adamw(rows + [[PTR + (1 << 16), PTR + (1 << 17), PTR + (1 << 16), 100, 0]]) == _lib.ERR_OPTIM_INPUT
    assert b"(states)" in lib.b200tp_last_error()


def test_addresses_of_many_tensors(lib):
    """The DLPack table of this torch, on host tensors: addresses of row-major tensors of the type and size, the first other one's index."""
    fn = _lib.tensor_rows()
    if fn is None:
        pytest.skip("this torch has no DLPack exchange table")
    good = [torch.zeros(3, 4), torch.nn.Parameter(torch.zeros(7)), torch.zeros(5)[2:], torch.zeros(0, 4), torch.zeros(()), torch.zeros(1, 6, 1),
            torch.zeros(6, 2)[:, :1][:4].t()[:, :1]]
    rows = np.zeros((len(good), 5), dtype=np.int64)
    rows[:, 3] = [t.numel() for t in good]

    def ask(tensors, dtype=0, device=-1, column=0):
        return fn(np.fromiter(map(id, tensors), np.int64, len(tensors)).ctypes.data, len(tensors), dtype, device, rows.ctypes.data, column)

    for column in (0, 1, 2):
        assert ask(good, column=column) == -1
        assert [p for p, t in zip(rows[:, column].tolist(), good) if t.numel()] == [t.data_ptr() for t in good if t.numel()]
    assert ask(good, dtype=1) == 0 and ask(good, device=0) == 0 and ask(good, column=3) == len(good)
    rows[:2, 3] = 12
    for bad in (torch.zeros(4, 3).t(), torch.zeros(3, 4, dtype=torch.bfloat16), torch.zeros(3, 4, dtype=torch.int32), torch.zeros(13),
                torch.zeros(3, 1).expand(3, 4), torch.zeros(24)[::2]):
        assert ask([good[0], bad]) == 1
    with pytest.raises(Exception):
        ask([torch.zeros(12).to_sparse()])
    assert ask([good[0].to(torch.bfloat16)], dtype=1) == -1


def test_exchange_tables_without_what_is_wanted(lib, monkeypatch):
    """A table that leaves the function out, or one of another version: tensors are then asked one by one.  The process's own
    prototypes stay as they are."""
    new = C.PYFUNCTYPE(C.py_object, C.c_void_p, C.c_char_p, C.c_void_p)(("PyCapsule_New", C.pythonapi))
    monkeypatch.setattr(C.pythonapi.PyCapsule_GetPointer, "restype", C.c_int)
    for version, entry in ((1, 0), (2, PTR), (1, PTR)):
        table = (C.c_uint64 * 8)(version, 0, 1, 1, 1, entry, 0, 0)
        monkeypatch.setattr(torch.Tensor, "__dlpack_c_exchange_api__", new(C.addressof(table), b"dlpack_exchange_api", None), raising=False)
        monkeypatch.setattr(_lib, "_tensor_rows", None)
        assert (_lib.tensor_rows() is None) == (version != 1 or not entry)
    assert C.pythonapi.PyCapsule_GetPointer.restype is C.c_int


def test_adamw_check_alone(lib):
    """Passes what would be launched, refuses what would be refused; with no GPU either way."""
    assert _adamw([ROW, [PTR + 400, PTR + 400, PTR + 400, 100, 256]], check_only=1) == _lib.OK
    assert _adamw([ROW, [PTR + 396, PTR + 400, PTR + 396, 100, 256]], check_only=1) == _lib.ERR_OPTIM_INPUT


def test_adamw_of_nothing(lib):
    assert _adamw([]) == _lib.OK


def _embedding(**change):
    a = _lib.EmbeddingArgs(PTR, 300, 1000, 64, 1, 1, 1.0, 64, -1)
    for k, v in change.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("change", [dict(ids=None), dict(n=-1), dict(n=(1 << 30) + 1), dict(v=0), dict(v=1 << 31), dict(d=0), dict(d=1 << 21),
                                    dict(dtype=2), dict(row_stride=-1)])
def test_embedding_arguments(lib, change):
    a = C.byref(_embedding(**change))
    assert lib.b200tp_embedding_bwd_workspace_bytes(a) == 0
    assert lib.b200tp_embedding_fwd(a, PTR, PTR, None, None) == _lib.ERR_EMBEDDING_INPUT
    assert lib.b200tp_embedding_bwd(a, PTR, PTR, PTR, 1 << 30, None, None) == _lib.ERR_EMBEDDING_INPUT


def test_embedding_pointers_and_workspace(lib):
    a = _embedding()
    need = lib.b200tp_embedding_bwd_workspace_bytes(C.byref(a))
    # keys and places twice, and two partial sums of a row for each window of 8 tokens at least
    assert 16 * 300 <= need <= 4 * 1280 + 2 * (38 * 64 * 4 + 256)
    assert lib.b200tp_embedding_bwd_workspace_bytes(C.byref(_embedding(n=64))) == 0       # up to 64 tokens: no sort
    bwd = lambda dy=PTR, dw=PTR, ws=PTR, n=need: lib.b200tp_embedding_bwd(C.byref(a), dy, dw, ws, n, None, None)
    assert bwd(dy=None) == bwd(dw=None) == bwd(dw=PTR + 8) == _lib.ERR_EMBEDDING_INPUT
    assert bwd(ws=None) == bwd(ws=PTR + 16) == bwd(n=need - 1) == _lib.ERR_WORKSPACE
    assert lib.b200tp_embedding_fwd(C.byref(a), None, PTR, None, None) == _lib.ERR_EMBEDDING_INPUT
    assert lib.b200tp_embedding_fwd(C.byref(_embedding(n=0, ids=None)), None, None, None, None) == _lib.OK


def test_status_text(lib):
    assert lib.b200tp_status_string(_lib.ERR_OPTIM_INPUT) == b"optimizer input error"
    assert lib.b200tp_status_string(_lib.ERR_EMBEDDING_INPUT) == b"embedding input error"
    with pytest.raises(EmbeddingInputError, match="outside the table"):
        _lib.raise_for_device_status(_lib.DEV_BAD_INDEX)


def test_forward_mode_derivatives_are_refused():
    """A dual tensor does not require a gradient, and its tangent must not vanish on the way."""
    from torch.autograd import forward_ad
    x, a = torch.zeros(2, 4), torch.zeros(2, 1)
    for leaf in (x, torch.zeros(2, 4, requires_grad=True)):
        with forward_ad.dual_level():
            dual = forward_ad.make_dual(leaf, torch.ones(2, 4))
            with pytest.raises(LossInputError, match="forward-mode"):
                preference_loss(dual)
            with pytest.raises(LossInputError, match="forward-mode"):
                policy_loss(dual, x, a)
            with pytest.raises(EmbeddingInputError, match="forward-mode"):
                embedding_lookup(torch.zeros(3, dtype=torch.int64), dual)
            with pytest.raises(LossInputError, match="CUDA"):       # a tensor without a tangent is looked at as ever
                preference_loss(x)


def test_host_tensors_are_refused():
    x, a = torch.zeros(2, 4), torch.zeros(2, 1)
    with pytest.raises(LossInputError, match="CUDA"):
        preference_loss(x)
    with pytest.raises(LossInputError, match="CUDA"):
        policy_loss(x, x, a)
    with pytest.raises(EmbeddingInputError, match="CUDA"):
        embedding_lookup(torch.zeros(3, dtype=torch.int64), x)
    with pytest.raises(OptimizerInputError, match="CUDA"):
        AdamWState.zeros([x])
    p = torch.nn.Parameter(x)
    p.grad = torch.zeros_like(x)
    with pytest.raises(OptimizerInputError, match="CUDA"):
        AdamW([p]).step()
