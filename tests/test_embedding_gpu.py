"""Embedding lookup and its table's gradient against their definitions in 64 bits, and its refusals.

Tolerances: a looked-up value is one fp32 product, rounded to the table's dtype: 2^-24 (fp32) or 2^-24 + 2^-8 (bf16) of the value.  A
gradient is a sum of k rows in fp32, each addition off by at most 2^-24 of the sum of magnitudes so far (k 2^-24 of all of them), then
one product and the store's rounding.
"""
import math

import pytest
import torch

from mlx_train_perf_b200 import DeviceTimeoutError, EmbeddingInputError, _lib, embedding_lookup
from mlx_train_perf_b200.core import loss
from mlx_train_perf_b200.core.loss import check_device_status, device_status

pytestmark = pytest.mark.gpu

E32 = 2.0 ** -24
STORE = {torch.float32: 0.0, torch.bfloat16: 2.0 ** -8}


def _ids(n, v, kind, g):
    if kind == "uniform":
        return torch.randint(0, v, (n,), generator=g)
    if kind == "words":                                            # about one over the rank, and a padded tail
        ids = (torch.exp(torch.rand(n, generator=g, dtype=torch.float64) * math.log(v + 1)).long() - 1).clamp(0, v - 1)
        ids[n - n // 4:] = v // 2
        return ids
    return torch.full((n,), v - 1)                                 # "one": every token the same


def _gradient_ref(ids, dy, v, scale, padding=None):
    """Sum and sum of magnitudes in 64 bits, and how many rows."""
    keep = (ids >= 0) & (ids < v) & (ids != (-1 if padding is None else padding))
    zeros = lambda: torch.zeros(v, dy.shape[1], dtype=torch.float64, device=dy.device)
    d = dy.double()[keep]
    count = torch.bincount(ids[keep], minlength=v).double()[:, None]
    return zeros().index_add_(0, ids[keep], d) * scale, zeros().index_add_(0, ids[keep], d.abs()) * abs(scale), count


def _check_gradient(got, ids, dy, v, scale, padding=None):
    want, size, count = _gradient_ref(ids, dy, v, scale, padding)
    off = (got.double() - want).abs() - (count + 1) * E32 * size - STORE[got.dtype] * want.abs() * (1 + 2.0 ** -8)
    assert not torch.isnan(got).any() and off.max().item() <= 1e-38, off.max().item()
    assert (got[(count == 0)[:, 0]] == 0).all()


def _check_lookup(got, ids, w, scale):
    want = w.double()[ids] * scale
    assert ((got.double() - want).abs() <= (2 * E32 + STORE[w.dtype] * (1 + 2.0 ** -8)) * want.abs()).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n,v,d,kind", [
    (1, 1, 1, "uniform"), (1, 1000, 64, "uniform"), (7, 3, 5, "uniform"), (60, 32768, 1024, "words"), (31, 511, 8, "uniform"),
    (8, 512, 2048, "one"), (9, 512, 2056, "one"), (257, 513, 67, "words"), (1000, 40, 2049, "words"), (4096, 7, 96, "uniform"),
    (16384, 151936, 128, "words"), (5000, 300000, 40, "uniform"), (70001, 1000, 72, "words"), (20000, 5, 520, "one"), (300, 70000, 4104, "uniform"),
    (256, 3000, 1024, "words"), (64, 9, 2056, "one"), (65, 9, 2056, "one"), (64, 20, 4100, "uniform"), (50, 70001, 67, "words"),
    (64, 40, 16384, "words"), (64, 40, 16392, "words"), (33, 8, 3, "uniform")])
def test_lookup_and_gradient(cuda_device, n, v, d, kind, dtype):
    dev = cuda_device
    g = torch.Generator().manual_seed(n + v)
    ids = _ids(n, v, kind, g).to(dev)
    w = torch.randn(v, d, generator=g).to(dtype).to(dev).requires_grad_(True)
    dy = torch.randn(n, d, generator=g).to(dtype).to(dev)
    scale = 1.0 if n % 2 else math.sqrt(d)
    out = embedding_lookup(ids, w, scale=scale)
    _check_lookup(out, ids, w.detach(), scale)
    if scale == 1.0:
        assert torch.equal(out, w.detach()[ids])
    grad, = torch.autograd.grad(out, w, dy, retain_graph=True)
    _check_gradient(grad, ids, dy, v, scale)
    assert torch.equal(grad, torch.autograd.grad(out, w, dy)[0])   # equal calls, equal bits
    check_device_status()


def test_gradient_is_exact_where_the_sums_are(cuda_device):
    """Whole numbers add up without rounding in any order: every row's sum, long runs across many windows among them, is exact, and a run
    of 100000 rows too."""
    dev = cuda_device
    g = torch.Generator().manual_seed(5)
    for n, v in ((5000, 37), (100000, 2), (100000, 30000)):
        ids = _ids(n, v, "words", g).to(dev)
        dy = torch.randint(-8, 9, (n, 24), generator=g).float().to(dev)
        w = torch.zeros(v, 24, device=dev, requires_grad=True)
        grad, = torch.autograd.grad(embedding_lookup(ids, w, scale=2.0), w, dy)
        assert torch.equal(grad.double(), _gradient_ref(ids, dy, v, 2.0)[0])


def test_gradient_against_differences(cuda_device):
    """The lookup is linear in its table: along any direction V, sum(dy * (f(W + V) - f(W))) is sum(dW * V), exactly where all values are
    whole numbers."""
    dev = cuda_device
    g = torch.Generator().manual_seed(6)
    whole = lambda *s: torch.randint(-6, 7, s, generator=g).float().to(dev)
    for n, v, d in ((50, 20, 24), (3000, 400, 72)):
        ids = _ids(n, v, "words", g).to(dev)
        w, way, dy = whole(v, d).requires_grad_(True), whole(v, d), whole(n, d)
        out = embedding_lookup(ids, w, scale=3.0)
        grad, = torch.autograd.grad(out, w, dy)
        moved = embedding_lookup(ids, w.detach() + way, scale=3.0)
        assert (dy.double() * (moved - out.detach()).double()).sum() == (grad.double() * way.double()).sum()


def test_order_of_the_sum_is_the_tokens_own(cuda_device):
    """Large and small values of one id: fp32 sums depend on the order, and the order is that of the tokens within a window (8 rows here,
    one id, one window)."""
    dev = cuda_device
    dy = torch.tensor([2.0 ** 24, 1.0, -2.0 ** 24, 1.0, 3.0], device=dev)[:, None].repeat(1, 16)
    w = torch.zeros(4, 16, device=dev, requires_grad=True)
    grad, = torch.autograd.grad(embedding_lookup(torch.full((5,), 2, device=dev), w), w, dy)
    acc = torch.zeros(16)
    for row in dy.cpu():
        acc = acc + row
    assert torch.equal(grad[2].cpu(), acc) and (grad[[0, 1, 3]] == 0).all()


def _sums_in_order(ids, dy, v, window):
    """Each row's sum in fp32 in the order that is promised beyond 64 tokens: tokens sorted by id, equal ids as they came; token by token
    within a window of sorted tokens; of a run that crosses windows the first window's sum, then the others', in four shares of
    adjacent windows whose sums are added in turn."""
    order = torch.argsort(ids, stable=True)
    out = torch.zeros(v, dy.shape[1])
    add = lambda rows: sum(rows[1:], rows[0]) if rows else torch.zeros(dy.shape[1])
    for key in ids.unique().tolist():
        at = (ids[order] == key).nonzero()[:, 0].tolist()          # adjacent places in the sorted order
        parts = {}
        for i in at:
            parts.setdefault(i // window, []).append(dy[order[i]])
        first, *others = [add(rows) for _, rows in sorted(parts.items())]
        each = (len(others) + 3) // 4
        shares = [others[k * each:(k + 1) * each] for k in range(4)]
        out[key] = add([add([first, *shares[0]]), *(add(s) for s in shares[1:])]) if others else first
    return out


@pytest.mark.parametrize("n,v,kind", [(65, 4, "uniform"), (65, 40, "uniform"), (72, 2, "uniform"), (200, 7, "words"), (700, 3, "one"), (1000, 60, "words"),
                                      (1000, 700, "words")])
def test_order_of_the_sum_beyond_64_tokens(cuda_device, n, v, kind):
    """Bit for bit, with values from 1 to 2^24 so that another order gives another sum: sort, windows of 8 tokens (as many as a thousand
    tokens take), and runs that cross them."""
    dev = cuda_device
    g = torch.Generator().manual_seed(n + v)
    ids = _ids(n, v, kind, g)
    dy = torch.randn(n, 16, generator=g) * 2.0 ** torch.randint(0, 25, (n, 16), generator=g)
    want = _sums_in_order(ids, dy, v, 8)
    assert not torch.equal(want, _sums_in_order(ids.flip(0), dy.flip(0), v, 8))    # the order shows
    w = torch.zeros(v, 16, device=dev, requires_grad=True)
    grad, = torch.autograd.grad(embedding_lookup(ids.to(dev), w), w, dy.to(dev))
    assert torch.equal(grad.cpu(), want)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_shapes_types_and_strides(cuda_device, dtype):
    dev = cuda_device
    g = torch.Generator().manual_seed(7)
    v, d = 300, 48
    w = torch.randn(v, d, generator=g).to(dtype).to(dev)
    for ids in (torch.tensor(5), torch.zeros(0, dtype=torch.int64), torch.zeros(0, 4, dtype=torch.int32), torch.randint(0, v, (2, 3, 5)),
                torch.randint(0, v, (4, 9), dtype=torch.int32), torch.randint(0, 100, (6,), dtype=torch.int16), torch.randint(0, v, (8, 10)).t()):
        ids = ids.to(dev)
        leaf = w.clone().requires_grad_(True)
        out = embedding_lookup(ids, leaf, scale=0.5)
        assert out.shape == (*ids.shape, d)
        _check_lookup(out.reshape(-1, d), ids.reshape(-1).long(), w, 0.5)
        dy = torch.randn(out.shape, generator=g).to(dtype).to(dev)
        out.backward(dy)
        _check_gradient(leaf.grad, ids.reshape(-1).long(), dy.reshape(-1, d), v, 0.5)
    # a table that is a slice of a wider one, at an odd column too; gradients that come transposed, expanded or sliced
    ids = torch.randint(0, v, (50,), generator=g).to(dev)
    wide = torch.randn(v, 100, generator=g).to(dtype).to(dev)
    for lo in (0, 8, 3):
        leaf = wide.clone().requires_grad_(True)
        out = embedding_lookup(ids, leaf[:, lo:lo + d])
        assert torch.equal(out, wide[ids, lo:lo + d])
        dy = torch.randn(50, 100, generator=g).to(dtype).to(dev)[:, lo:lo + d]
        out.backward(dy)
        _check_gradient(leaf.grad[:, lo:lo + d], ids, dy, v, 1.0)
    for make in (lambda: torch.randn(d, 50, generator=g).to(dtype).to(dev).t(), lambda: torch.ones(1, 1, dtype=dtype, device=dev).expand(50, d),
                 lambda: torch.randn(1, d, generator=g).to(dtype).to(dev).expand(50, d)):
        leaf, dy = w.clone().requires_grad_(True), make()
        embedding_lookup(ids, leaf).backward(dy)
        _check_gradient(leaf.grad, ids, dy, v, 1.0)
    t = torch.randn(d, v, generator=g).to(dtype).to(dev).t()
    assert torch.equal(embedding_lookup(ids, t), t[ids])


def test_padding_and_ids_outside_the_table(cuda_device):
    dev = cuda_device
    g = torch.Generator().manual_seed(9)
    v, d = 64, 32
    w = torch.randn(v, d, generator=g).to(dev).requires_grad_(True)
    ids = torch.randint(0, v, (500,), generator=g).to(dev)
    dy = torch.randn(500, d, generator=g).to(dev)
    for padding in (0, 63, -1):
        out = embedding_lookup(ids, w, padding_idx=padding)
        assert torch.equal(out, w.detach()[ids])
        grad, = torch.autograd.grad(out, w, dy)
        _check_gradient(grad, ids, dy, v, 1.0, padding % v)
        assert (grad[padding] == 0).all()
    check_device_status()
    wild = ids.clone()
    wild[::7] = torch.tensor([-1, v, 2 ** 40, -2 ** 62], device=dev).repeat(18)
    out = embedding_lookup(wild, w)
    assert (out[::7] == 0).all()
    grad, = torch.autograd.grad(out, w, dy)
    _check_gradient(grad, wild, dy, v, 1.0)
    with pytest.raises(EmbeddingInputError, match="outside"):
        check_device_status()
    check_device_status()                                          # reported once
    with pytest.raises(EmbeddingInputError, match="0 <= id < V"):
        embedding_lookup(wild, w, validate_ids=True)
    embedding_lookup(ids, w, validate_ids=True)


def test_a_bad_id_does_not_hide_a_wait_that_ran_out(cuda_device):
    """Both in one step, the bad id first (the wait is the library's self-test, which runs into its limit): both are reported, the wait
    before the id, each once."""
    dev = cuda_device
    check_device_status()
    embedding_lookup(torch.tensor([3, 99], device=dev), torch.zeros(10, 8, device=dev))
    waited = torch.zeros(2, dtype=torch.int64, device=dev)
    _lib.check(_lib.load().b200tp_selftest_bounded_wait(waited.data_ptr(), torch.cuda.current_stream(dev).cuda_stream,
                                                        device_status(dev).data_ptr()))
    with pytest.raises(DeviceTimeoutError):
        check_device_status()
    with pytest.raises(EmbeddingInputError, match="outside"):
        check_device_status(dev)
    check_device_status()


def test_a_bad_id_of_the_first_call_in_inference_mode(cuda_device, monkeypatch):
    """The words that are made in that call can be read and cleared outside it."""
    for words in ("_status", "_index_status"):
        monkeypatch.setattr(loss, words, {})
    with torch.inference_mode():
        embedding_lookup(torch.tensor([3, 99], device=cuda_device), torch.zeros(10, 8, device=cuda_device))
    with pytest.raises(EmbeddingInputError, match="outside"):
        check_device_status()
    check_device_status()


def test_values_that_are_not_finite_stay_in_their_rows(cuda_device):
    dev = cuda_device
    w = torch.zeros(40, 16, device=dev, requires_grad=True)
    ids = torch.arange(100, device=dev) % 40
    dy = torch.ones(100, 16, device=dev)
    dy[3, 2], dy[45, 7] = math.nan, math.inf
    grad, = torch.autograd.grad(embedding_lookup(ids, w), w, dy)
    assert torch.isnan(grad[3, 2]) and torch.isinf(grad[5, 7])
    grad[3, 2] = grad[5, 7] = 0.0
    want = torch.bincount(ids, minlength=40).float()[:, None].repeat(1, 16)
    want[3, 2] = want[5, 7] = 0.0
    assert torch.equal(grad, want)


def test_without_gradients_and_second_derivative(cuda_device):
    dev = cuda_device
    w = torch.randn(10, 8, device=dev, requires_grad=True)
    ids = torch.tensor([1, 2, 1], device=dev)
    with torch.no_grad():
        assert not embedding_lookup(ids, w).requires_grad
    assert not embedding_lookup(ids, w.detach()).requires_grad
    with pytest.raises(EmbeddingInputError, match="second derivative"):
        torch.autograd.grad(embedding_lookup(ids, w).square().sum(), w, create_graph=True)


def test_offsets_beyond_32_bits(cuda_device):
    """A table and a batch of more than 2^31 elements: rows at both ends, forward and backward."""
    dev = cuda_device
    d, v = 4096, (1 << 31) // 4096 + 7
    w = torch.zeros(v, d, dtype=torch.bfloat16, device=dev)
    w[-1], w[-5], w[1] = 3.0, 5.0, 7.0
    w.requires_grad_(True)
    ids = torch.tensor([v - 1, 1, v - 5, v - 1], device=dev)
    out = embedding_lookup(ids, w)
    assert out[:, 0].tolist() == [3.0, 7.0, 5.0, 3.0]
    grad, = torch.autograd.grad(out, w, torch.ones_like(out))
    assert grad[-1, -1] == 2 and grad[-5, 0] == 1 and grad[1, 9] == 1 and grad.abs().sum(dtype=torch.float64).item() == 4 * d
    del w, grad, out
    n = (1 << 31) // 4096 + 9
    w = torch.arange(1, 4, dtype=torch.bfloat16, device=dev)[:, None].repeat(1, d).requires_grad_(True)
    ids = torch.zeros(n, dtype=torch.int64, device=dev)
    ids[-1], ids[-2] = 2, 1
    out = embedding_lookup(ids, w)
    assert out[-1, 0] == 3 and out[-2, -1] == 2 and out[0, 0] == 1
    dy = torch.zeros_like(out)
    dy[-1], dy[-2], dy[-3], dy[0] = 4.0, 8.0, 16.0, 32.0
    grad, = torch.autograd.grad(out, w, dy)
    assert (grad[2] == 4).all() and (grad[1] == 8).all() and (grad[0] == 48).all()


def test_other_stream_and_captured(cuda_device):
    dev = cuda_device
    g = torch.Generator().manual_seed(11)
    w = torch.randn(500, 64, generator=g).to(dev).requires_grad_(True)
    ids, more = (torch.randint(0, 500, (2, 700), generator=g)).to(dev)
    dy = torch.randn(700, 64, generator=g).to(dev)

    def both(i):
        out = embedding_lookup(i, w, scale=2.0)
        return out.detach(), torch.autograd.grad(out, w, dy)[0]

    want = [both(i) for i in (ids, more)]
    static = ids.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = [both(static) for _ in range(3)]
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for k in got for a, b in zip(k, want[0]))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = both(static)
    for k, i in enumerate((more, ids)):
        static.copy_(i)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want[1 - k]))


def test_refusals(cuda_device):
    dev = cuda_device
    w = torch.zeros(10, 8, device=dev)
    ids = torch.tensor([1, 2], device=dev)
    for k, call in enumerate([
            lambda: embedding_lookup(ids, w[0]), lambda: embedding_lookup(ids, w.half()), lambda: embedding_lookup(ids.float(), w),
            lambda: embedding_lookup(ids.bool(), w), lambda: embedding_lookup(ids.cpu(), w), lambda: embedding_lookup(ids, w[:0]),
            lambda: embedding_lookup(ids, w[:, :0]), lambda: embedding_lookup(ids, w, padding_idx=10), lambda: embedding_lookup(ids, w, padding_idx=-11),
            lambda: embedding_lookup(ids.cpu(), w.cpu())]):
        with pytest.raises(EmbeddingInputError):
            call()
            pytest.fail(f"call {k} was not refused")
