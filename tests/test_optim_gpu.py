"""The AdamW step against its definition in 64 bits, the layout of its states, and the optimizer around it.

Tolerances count roundings of 2^-24 (half a step of fp32).  m: two factors rounded to fp32 (b1, 1 - b1), a product and a fused sum: 4 of
|b1 m| + |c1 g|; v: 5 of b2 v + c2 g^2.  The update lr/bc1 m / (sqrt(v) bc2 + eps): what m is off by over the denominator, and
4 (v under the root: half of 5, the root 2 with its Newton step) + 2 (bc2, eps) + 4 (reciprocal or quotient: 2 ulps) + 3 (rate, products)
of its own, rounded up to 16.  p: 3 of |p| (decay, product, sum).  A stored bf16 value is off by another 2^-8.
8-bit: a stored m is half an e4m3 step off (2^-4 of the value, or 2^-10 scales below 2^-6), a stored root one step at most.
"""
import copy
import math

import pytest
import torch

from mlx_train_perf_b200 import AdamW, AdamWState, OptimizerInputError, adamw_step

pytestmark = pytest.mark.gpu

E32 = 2.0 ** -24
RULE = dict(lr=3e-3, betas=(0.9, 0.99), eps=1e-6, weight_decay=0.05)


def _tensors(shapes, dtype, dev, seed, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return [(torch.randn(s, generator=g) * scale).to(dtype).to(dev) for s in shapes]


def _fill(state, seed):
    """Moments in the middle of a run, by steps on random gradients."""
    g = torch.Generator(device=state.exp_avg.device).manual_seed(seed)
    dev = state.exp_avg.device
    for t in range(3):
        params = [torch.zeros(n, device=dev) for n in state.numels]
        grads = [torch.randn(n, generator=g, device=dev) * 0.1 for n in state.numels]
        master, state.master = state.master, None
        adamw_step(params, grads, state, lr=0.0, betas=(0.9, 0.99))
        state.master = master


def _ref(p, g, m, v, step, grad_scale=1.0, *, lr, betas, eps, weight_decay):
    """New p, m, v in 64 bits, and how far each may be off."""
    p, g, m, v = p.double().reshape(-1), g.double().reshape(-1) * grad_scale, m.double(), v.double()
    b1, b2 = betas
    m1, v1 = b1 * m + (1 - b1) * g, b2 * v + (1 - b2) * g * g
    tm, tv = 4 * E32 * (b1 * m.abs() + (1 - b1) * g.abs()), 5 * E32 * v1
    denom = (v1 / (1 - b2 ** step)).sqrt() + eps
    rate = lr / (1 - b1 ** step)
    p1 = p * (1 - lr * weight_decay) - rate * m1 / denom
    tp = rate * tm / denom + 16 * E32 * (rate * m1 / denom).abs() + 3 * E32 * p.abs()
    return p1, m1, v1, tp, tm, tv


def _assert_within(got, want, tol, store=0.0):
    off = (got.double().reshape(-1) - want).abs() - tol - store * want.abs() - 1e-37
    assert not torch.isnan(got.float()).any() and (off.max().item() if off.numel() else 0.0) <= 0.0, off.max().item()


def _e4m3_step(y):
    """Distance of the e4m3 values around y."""
    return 2.0 ** (torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6))) - 3)


def _check_moments(state, i, m1, v1, tm, tv):
    m, v = state.moments(i)
    if state.bits == 32:
        _assert_within(m, m1, tm)
        _assert_within(v, v1, tv)
        return
    scales = state.view("scales", i).double().repeat_interleave(256, 0)[:m.numel()]
    zero = torch.zeros(m.numel(), dtype=torch.float64, device=m.device)
    sm, sr = scales[:, 0], scales[:, 1]
    _assert_within(m, m1, torch.where(sm > 0, 0.5 * _e4m3_step(m1 / sm.clamp(min=1e-300)) * sm, zero) * (1 + 64 * E32) + 2 * tm + 1e-29)
    r1 = v1.sqrt()
    step = torch.where(sr > 0, _e4m3_step(r1 / sr.clamp(min=1e-300)) * sr, zero)
    _assert_within(v.sqrt(), r1, step * (1 + 64 * E32) + 16 * E32 * r1)
    # a block's scales: its largest values over 448 (codes of the largest values are 448, or 416 where a dither went down)
    n, blocks = m.numel(), state.view("scales", i)
    pad = torch.zeros(blocks.shape[0] * 256, dtype=torch.float64, device=m.device)
    for col, x in ((0, m1.abs()), (1, r1)):
        pad.zero_()[:n] = x
        torch.testing.assert_close(blocks[:, col].double(), pad.reshape(-1, 256).amax(1) / 448, rtol=32 * E32, atol=1e-32)
    assert ((v > 0) == (v1 > 1e-30)).all()


SHAPES = [(1,), (255,), (256,), (257,), (3, 5, 7), (4096,), (0,), (64, 129), (20011,)]


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("p_dtype,g_dtype,master", [(torch.float32, torch.float32, False), (torch.float32, torch.bfloat16, False),
                                                    (torch.bfloat16, torch.bfloat16, False), (torch.bfloat16, torch.float32, False),
                                                    (torch.bfloat16, torch.bfloat16, True), (torch.bfloat16, torch.float32, True)])
@pytest.mark.parametrize("scale", [1.0, 0.125])
def test_step(cuda_device, bits, p_dtype, g_dtype, master, scale):
    dev = cuda_device
    params, grads = _tensors(SHAPES, p_dtype, dev, 1), _tensors(SHAPES, g_dtype, dev, 2, 0.2)
    state = AdamWState.zeros(params, bits=bits, master=master)
    _fill(state, 5)
    before = [tuple(t.clone() for t in state.moments(i)) for i in range(len(SHAPES))]
    values = [(state.view("master", i) if master else p.reshape(-1)).clone() for i, p in enumerate(params)]
    assert state.steps == [3] * len(SHAPES)
    how = torch.tensor([scale], device=dev) if scale != 1.0 else 1.0
    adamw_step(params, grads, state, grad_scale=how, **RULE)
    assert state.steps == [4] * len(SHAPES)
    for i, (p, g) in enumerate(zip(params, grads)):
        p1, m1, v1, tp, tm, tv = _ref(values[i], g, *before[i], 4, scale, **RULE)
        _assert_within(p, p1, tp, 2.0 ** -8 * (1 + 2.0 ** -16) if p_dtype == torch.bfloat16 else 0.0)
        if master:
            _assert_within(state.view("master", i), p1, tp)
            assert torch.equal(p.reshape(-1), state.view("master", i).to(torch.bfloat16))
        _check_moments(state, i, m1, v1, tm, tv)
    # what lies behind each tensor in the states stays zero
    for name in ("exp_avg", "exp_avg_sq") + (("master",) if master else ()):
        flat = getattr(state, name).float()
        for i in range(len(SHAPES)):
            o, n = int(state.rows[i, 4]), state.numels[i]
            assert (flat[o + n:o + (n + 255) // 256 * 256] == 0).all()


@pytest.mark.parametrize("bits", [32, 8])
def test_what_lies_behind_a_tensor_stays_zero_without_eps(cuda_device, bits):
    """0 / (0 + 0) of elements that are not there must not get into the masters' padding."""
    params, grads = _tensors(SHAPES, torch.bfloat16, cuda_device, 1), _tensors(SHAPES, torch.bfloat16, cuda_device, 2)
    state = AdamWState.zeros(params, bits=bits, master=True)
    for _ in range(2):
        adamw_step(params, grads, state, lr=0.1, eps=0.0)
    for i, n in enumerate(state.numels):
        o = int(state.rows[i, 4])
        for flat in (state.master, state.exp_avg, state.exp_avg_sq):
            assert (flat[o + n:o + (n + 255) // 256 * 256].float() == 0).all()
    assert torch.isfinite(state.master).all()


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("master", [False, True])
def test_other_buffers_get_what_the_step_in_place_gives(cuda_device, bits, master):
    dev = cuda_device
    params, grads = _tensors(SHAPES, torch.bfloat16, dev, 3), _tensors(SHAPES, torch.bfloat16, dev, 4)
    state = AdamWState.zeros(params, bits=bits, master=master)
    _fill(state, 6)
    names = [n for n in ("exp_avg", "exp_avg_sq", "scales", "master") if getattr(state, n) is not None]
    kept = {n: getattr(state, n).clone() for n in names}
    old = [p.clone() for p in params]
    to = [torch.full_like(p, float("nan")) for p in params]
    after = AdamWState.zeros(params, bits=bits, master=master)
    adamw_step(params, grads, state, step=9, out=(to, after), **RULE)
    assert all(torch.equal(p, q) for p, q in zip(params, old)) and state.steps == [3] * len(SHAPES) and after.steps == [9] * len(SHAPES)
    assert all(torch.equal(getattr(state, n).view(torch.uint8), kept[n].view(torch.uint8)) for n in names)
    adamw_step(params, grads, state, step=9, **RULE)
    assert all(torch.equal(p, q) for p, q in zip(params, to))
    assert all(torch.equal(getattr(state, n).view(torch.uint8), getattr(after, n).view(torch.uint8)) for n in names)


def test_other_buffers_are_known_to_have_changed(cuda_device):
    """A graph that saved an output's old value must not use the new one."""
    p, to = torch.ones(300, device=cuda_device), torch.ones(300, device=cuda_device, requires_grad=True)
    loss = to.square().sum()
    adamw_step([p], [p.clone()], AdamWState.zeros([p]), out=([to], AdamWState.zeros([p])), **RULE)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()


@pytest.mark.parametrize("bits", [32, 8])
def test_a_gradient_that_its_own_result_replaces(cuda_device, bits):
    dev = cuda_device
    params, grads = _tensors(SHAPES, torch.bfloat16, dev, 3), _tensors(SHAPES, torch.bfloat16, dev, 4)
    one, two = AdamWState.zeros(params, bits=bits), AdamWState.zeros(params, bits=bits)
    over = [g.clone() for g in grads]
    adamw_step(params, over, one, out=(over, two), **RULE)
    adamw_step(params, grads, one, **RULE)
    assert all(torch.equal(p, q) for p, q in zip(params, over))


@pytest.mark.parametrize("bits", [32, 8])
def test_unaligned_views_and_strided_gradients(cuda_device, bits):
    """Parameters and gradients one element off an aligned address, odd sizes, gradients transposed: the values of aligned ones."""
    dev = cuda_device
    sizes = [(3, 301), (17, 1000), (4099,)]
    got = []
    for off in (0, 1):
        params = [torch.empty(math.prod(s) + 8, dtype=torch.bfloat16, device=dev)[off:off + math.prod(s)].view(s).copy_(t)
                  for s, t in zip(sizes, _tensors(sizes, torch.bfloat16, dev, 7))]
        grads = [torch.empty(math.prod(s) + 8, dtype=torch.bfloat16, device=dev)[off:off + math.prod(s)].view(s).copy_(t)
                 for s, t in zip(sizes, _tensors(sizes, torch.bfloat16, dev, 8))]
        if off:
            grads[0] = grads[0].t().contiguous().t()
        around = [p._base[-8 + off:].clone() for p in params]
        state = AdamWState.zeros(params, bits=bits)
        adamw_step(params, grads, state, **RULE)
        adamw_step(params, grads, state, **RULE)
        assert all(torch.equal(p._base[-8 + off:].view(torch.int16), a.view(torch.int16)) for p, a in zip(params, around))
        got.append([*(p.clone() for p in params), state.exp_avg.view(torch.uint8), state.exp_avg_sq.view(torch.uint8)])
    assert all(torch.equal(a, b) for a, b in zip(*got))


def test_more_tensors_than_one_launch_takes(cuda_device):
    dev = cuda_device
    for count in (48, 49, 600, 601, 1300):
        params = [torch.full((1 + k % 3,), float(k), device=dev) for k in range(count)]
        grads = [torch.full((1 + k % 3,), 0.5 - k % 2, device=dev) for k in range(count)]
        state = AdamWState.zeros(params)
        adamw_step(params, grads, state, lr=0.25, weight_decay=0.0, eps=0.0)
        for k, p in enumerate(params):            # the first step moves by lr against the gradient's sign
            assert (p - (k + (0.25 if k % 2 else -0.25))).abs().max().item() <= 4e-7 * max(1, k), k


def test_tensors_without_gradients_and_of_different_ages(cuda_device):
    dev = cuda_device
    shapes = [(300,), (5,), (1000,)]
    params, grads = _tensors(shapes, torch.float32, dev, 9), _tensors(shapes, torch.float32, dev, 10)
    state = AdamWState.zeros(params)
    alone = [AdamWState.zeros([p]) for p in params]
    single = [p.clone() for p in params]
    for which in ((0, 1, 2), (0, 2), (1,), (), (0, 1, 2)):
        adamw_step(params, [g if i in which else None for i, g in enumerate(grads)], state, **RULE)
        for i in which:
            adamw_step([single[i]], [grads[i]], alone[i], **RULE)
    assert state.steps == [3, 3, 3] and all(torch.equal(p, q) for p, q in zip(params, single))
    adamw_step(params, [grads[0], None, None], state, **RULE)
    assert state.steps == [4, 3, 3]
    adamw_step(params, grads, state, **RULE)                      # two ages in one call
    for i in ([0, 0], [1], [2]):
        for k in i:
            adamw_step([single[k]], [grads[k]], alone[k], **RULE)
    assert state.steps == [5, 4, 4] and all(torch.equal(p, q) for p, q in zip(params, single))


def test_a_strided_gradient_before_a_missing_one(cuda_device):
    dev = cuda_device
    params = _tensors([(6, 50), (40,), (7, 9)], torch.float32, dev, 11)
    same = [p.clone() for p in params]
    g = _tensors([(50, 6), (40,), (9, 7)], torch.float32, dev, 12)
    state, other = AdamWState.zeros(params), AdamWState.zeros(params)
    adamw_step(params, [g[0].t(), None, g[2].t()], state, **RULE)
    adamw_step(same, [g[0].t().contiguous(), g[1], g[2].t().contiguous()], other, **RULE)
    assert torch.equal(params[0], same[0]) and torch.equal(params[2], same[2]) and not torch.equal(params[1], same[1])
    assert state.steps == [1, 0, 1]
    with pytest.raises(OptimizerInputError, match="dense"):
        adamw_step(params[:2], [g[0].t(), g[1].to_sparse()], AdamWState.zeros(params[:2]), **RULE)


def test_tensors_asked_one_by_one(cuda_device, monkeypatch):
    """Without the DLPack table (another torch), or with a tensor class of its own: the same step, the same refusals."""
    from mlx_train_perf_b200 import _lib

    class Own(torch.Tensor):
        pass

    dev = cuda_device
    params, grads = _tensors([(6, 50), (40,)], torch.bfloat16, dev, 13), _tensors([(6, 50), (40,)], torch.bfloat16, dev, 14)
    want = [p.clone() for p in params]
    adamw_step(want, grads, AdamWState.zeros(want), **RULE)
    own = [p.clone().as_subclass(Own) for p in params]
    adamw_step(own, grads, AdamWState.zeros(own), **RULE)
    assert all(torch.equal(a.as_subclass(torch.Tensor), b) for a, b in zip(own, want))
    monkeypatch.setattr(_lib, "tensor_rows", lambda: None)
    state = AdamWState.zeros(params)
    for bad in ([grads[0], grads[1].float()], [grads[0], grads[1].cpu()], [grads[0], grads[1][:39]], [grads[0].half(), grads[1].half()]):
        with pytest.raises(OptimizerInputError):
            adamw_step(params, bad, state, **RULE)
    with pytest.raises(OptimizerInputError):
        adamw_step([params[0].t(), params[1]], grads, state, **RULE)
    adamw_step(params, grads, state, **RULE)
    assert all(torch.equal(a, b) for a, b in zip(params, want))


def test_8_bit_codes_are_off_by_three_roundings_at_most(cuda_device):
    """A scale is the largest times 1/448, each of the two rounded, and a code is m over it, rounded: where the exact quotient is farther than
    3 x 2^-24 of itself (and what the three multiply to, 2^-6 of that) from the middle between two codes, the code is the nearest one.
    With betas of 0 the first step's m are the gradients themselves, placed around such middles here."""
    dev = cuda_device
    g = torch.Generator().manual_seed(31)
    blocks = 8192
    top = 1 + torch.rand(blocks, 1, generator=g)
    middle = (torch.randint(8, 15, (blocks, 256), generator=g) + 0.5) * 2.0 ** torch.randint(-8, 5, (blocks, 256), generator=g)
    near = 1 + torch.randint(-64, 65, (blocks, 256), generator=g).double() / 16 * E32
    grad = (middle.double() * near * top.double() / 448).float()
    grad[:, :1] = top
    p = [torch.zeros(blocks * 256, device=dev)]
    state = AdamWState.zeros(p, bits=8)
    adamw_step(p, [grad.reshape(-1).to(dev)], state, lr=0.0, betas=(0.0, 0.0))
    got = state.exp_avg.cpu().float().double().reshape(blocks, 256)[:, 1:]
    y, middle = (grad.double() * 448 / top.double())[:, 1:], middle.double()[:, 1:]
    nearest = torch.round(y / _e4m3_step(y)) * _e4m3_step(y)
    clear = (y / middle - 1).abs() > 3 * E32 * (1 + 2.0 ** -6)
    assert 0.1 < clear.double().mean() < 0.5
    assert torch.equal(got[clear], nearest[clear])


def _mixed_bits(n, step, dev, complement=False):
    """For each of n positions 16 bits of a 32-bit mix of its pair (or the pair's complement) and the step, times 16 and 8."""
    x = torch.arange(n // 2, device=dev)
    x = ((x ^ 0xFFFFFFFF) if complement else x) + step * 0x3504F333
    x = (x * 0x1E3779B1) & 0xFFFFFFFF
    x = ((x ^ (x >> 16)) * 0x7FEB352D) & 0xFFFFFFFF
    x = ((x ^ (x >> 15)) * 0x046CA68B) & 0xFFFFFFFF
    x = x ^ (x >> 16)
    return torch.stack([x & 0xFFFF, x >> 16], dim=-1).reshape(-1) * 16 + 8


def _by_dither(y, d):
    """y >= 0 to the e4m3 value below or above it, exactly: floor of y over the distance of values there, plus the dither."""
    step = _e4m3_step(y.double())
    return ((y.double() / step + d.double() / 2 ** 20).floor() * step).float()


@pytest.mark.parametrize("betas", [(0.9, 0.999), (0.5, 0.9), (0.95, 0.95), (0.99, 0.999)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("grad_scale", [1.0, 0.3])
def test_8_bit_moments_are_those_of_fp32_operations(cuda_device, betas, dtype, grad_scale):
    """Bit for bit: moments, scales and codes of two million elements by elementary fp32 operations, each rounded by itself.  (Sums of a
    dither and a value are exact here and rounded in fp32 there: some 2^-20 of the 20000 values below 2^-6.)"""
    dev, n, step = cuda_device, 1 << 21, 7
    g = torch.Generator(device=dev).manual_seed(17)
    normal = lambda: torch.randn(n, generator=g, device=dev)
    size = torch.exp(torch.randn(n // 256, 1, generator=g, device=dev)).expand(-1, 256).reshape(-1) * 1e-3
    grad = (normal() * size).to(dtype)
    m8, r8 = (normal() * 120).clamp(-448, 448), (normal().abs() * 100 + 1).clamp(max=448).to(torch.float8_e4m3fn)
    m8[::97], grad[::97] = torch.randint(-15, 16, (m8[::97].numel(),), generator=g, device=dev) / 512, grad[::97] * 1e-5    # fed by little
    m8 = m8.to(torch.float8_e4m3fn)
    scales = torch.rand(n // 256, 2, generator=g, device=dev) * 1e-5 + 1e-6
    state = AdamWState([n], m8.clone(), r8.clone(), scales=scales.clone())
    adamw_step([torch.zeros(n, dtype=dtype, device=dev)], [grad], state, lr=1e-3, betas=betas, step=step, grad_scale=grad_scale)
    rows = lambda t: t.reshape(-1, 256)
    one = lambda v: torch.tensor(v, dtype=torch.float32, device=dev)
    (b1, b2), a = betas, grad.float() * one(grad_scale)
    old_m, old_r = (rows(m8.float()) * scales[:, :1]).reshape(-1), (rows(r8.float()) * scales[:, 1:]).reshape(-1)
    fed = a * one(1 - b1)
    m, v = old_m * one(b1) + fed, old_r * old_r * one(b2) + a * one(1 - b2) * a
    r = v.sqrt()
    want = torch.stack([rows(m).abs().amax(1), r.reshape(-1, 256).amax(1)], dim=1) * one(1 / 448)
    assert torch.equal(state.scales, want)
    x, y = (rows(m) / want[:, :1]).reshape(-1), (rows(r) / want[:, 1:]).reshape(-1)
    small = (m8.float().abs() < 2.0 ** -6) & (fed.abs() < 2.0 ** -6 * scales[:, :1].expand(-1, 256).reshape(-1))
    dithered = _by_dither(x.abs(), _mixed_bits(n, step, dev, complement=True)).copysign(x)
    codes_m = torch.where(small | (b1 > 0.9), dithered, x).clamp(-448, 448).to(torch.float8_e4m3fn)
    codes_r = _by_dither(y, _mixed_bits(n, step, dev)).clamp(2.0 ** -9, 448).to(torch.float8_e4m3fn)
    for got, codes, value in ((state.exp_avg, codes_m, x), (state.exp_avg_sq, codes_r, y)):
        off = got.view(torch.uint8) != codes.view(torch.uint8)
        assert not off[value.abs() >= 2.0 ** -6].any() and off.sum() <= 1
    assert 5000 < small.sum() < 25000


def test_8_bit_roots_are_rounded_without_drift(cuda_device):
    """A million equal roots between two codes: the mean of the codes is the root, up to five standard errors and the dither's own
    2^-17 of a step; and a v that is not zero never becomes zero, whatever the block's largest."""
    dev = cuda_device
    n = 1 << 20
    p = [torch.zeros(n, device=dev)]
    g = torch.full((n,), 1.3, device=dev)
    g[::256] = 7.0                                                # the blocks' scale
    state = AdamWState.zeros(p, bits=8)
    adamw_step(p, [g], state, lr=0.0, betas=(0.0, 0.0))
    roots = state.moments(0)[1].sqrt().double().reshape(-1, 256)[:, 1:]
    step = 2.0 ** (math.floor(math.log2(1.3 / (7.0 / 448))) - 3) * 7.0 / 448
    se = step / 2 / math.sqrt(roots.numel())
    assert roots.unique().numel() == 2 and abs(roots.mean().item() - 1.3) < 5 * se + step * 2.0 ** -17 + 1.3 * 8 * E32
    # the same step again gives the same codes, the next one others
    again = AdamWState.zeros(p, bits=8)
    adamw_step(p, [g], again, lr=0.0, betas=(0.0, 0.0))
    assert torch.equal(again.exp_avg_sq.view(torch.uint8), state.exp_avg_sq.view(torch.uint8))
    adamw_step(p, [g], again, lr=0.0, betas=(0.0, 0.0))
    assert not torch.equal(again.exp_avg_sq.view(torch.uint8), state.exp_avg_sq.view(torch.uint8))
    g = torch.full((n,), 1e-12, device=dev)
    g[::256] = 1e6
    g[1::256] = 0.0
    adamw_step(p, [g], state, lr=0.0, betas=(0.0, 0.0))
    v = state.moments(0)[1].reshape(-1, 256)
    assert (v[:, 1] == 0).all() and (v[:, 2:] > 0).all() and (v[:, 0] > 0).all()


@pytest.mark.parametrize("beta1,code", [(0.9, 4), (0.9, -4), (0.9, 1), (0.95, 9), (0.95, -9), (0.99, 8), (0.99, 300), (0.95, 3)])
def test_8_bit_m_that_nothing_feeds_is_not_held(cuda_device, beta1, code):
    """Half a million equal m without a gradient, each a code (in units of 2^-9 up to 7, of 2^-6 / 8 ... above) that rounding to nearest
    would bring back: after a step their mean is beta1 times the code, up to five standard errors, the dither's own 2^-17 of a
    distance and the roundings of m and of its scale."""
    dev = cuda_device
    n = 256 * 2048
    y = torch.tensor(code / 512.0).to(torch.float8_e4m3fn).float().item()
    m = torch.full((n,), y, device=dev)
    m[::256] = 448.0
    state = AdamWState([n], m.to(torch.float8_e4m3fn), torch.full((n,), 1.0, device=dev).to(torch.float8_e4m3fn),
                       scales=torch.ones(n // 256, 2, device=dev), steps=[200])
    g = torch.zeros(n, device=dev)
    g[::256] = 448.0                                              # holds the scale
    adamw_step([torch.zeros(n, device=dev)], [g], state, lr=0.0, betas=(beta1, 0.999))
    got = state.moments(0)[0].double().reshape(-1, 256)[:, 1:]
    step = _e4m3_step(torch.tensor(y)).item()
    se = step / 2 / math.sqrt(got.numel())
    assert 1 <= got.unique().numel() <= 2 and got.unique().abs().min() < abs(y)
    assert abs(got.mean().item() - beta1 * y) < 5 * se + step * 2.0 ** -17 + abs(y) * 8 * E32


@pytest.mark.parametrize("betas,steps", [((0.9, 0.999), 4000), ((0.9, 0.95), 3000), ((0.95, 0.95), 3000), ((0.95, 0.999), 3000)])
def test_8_bit_parameters_stop_where_gradients_do(cuda_device, betas, steps):
    """Twenty steps with gradients of 0.5, then none, while the block's largest stays at 1: a parameter moves as far as in 64 bits.  What may
    differ: m rounded to nearest falls by at least two thirds of what it should a step (code 15 goes to 14 and not to 13.5, 14
    to 13 and not to 12.6), dithered m by as much in the mean; 1 / sqrt(v) is up to 1.18 times too large in the mean (a
    root's dither has a variance of at most (1/8)^2 / 4 a step, weighed with the decay of m / sqrt(v), 0.975 a step at the
    slowest).  So 0.95 to 1.8 times; m is zero at the end (beta1^t is below 1e-60), and nothing moves any more."""
    dev = cuda_device
    n = 256 * 64
    p, state = [torch.zeros(n, device=dev)], AdamWState.zeros([torch.zeros(n, device=dev)], bits=8)
    hot = torch.zeros(n, device=dev)
    hot[::256] = 1.0
    fed = torch.where(hot > 0, 1.0, 0.5)
    want = m = v = 0.0
    for t in range(1, steps + 1):
        g = 0.5 if t <= 20 else 0.0
        m, v = betas[0] * m + (1 - betas[0]) * g, betas[1] * v + (1 - betas[1]) * g * g
        want += m / (1 - betas[0] ** t) / math.sqrt(v / (1 - betas[1] ** t)) if v > 0 else 0.0
        adamw_step(p, [fed if t <= 20 else hot], state, lr=1.0, betas=betas, eps=0.0, weight_decay=0.0)
    rest = hot == 0
    moved = -p[0][rest].double()
    assert 0.95 * want < moved.mean().item() < 1.8 * want, (moved.mean().item(), want)
    assert (state.moments(0)[0][rest] == 0).all()
    before = p[0].clone()
    adamw_step(p, [hot], state, lr=1.0, betas=betas, eps=0.0, weight_decay=0.0)
    assert torch.equal(p[0][rest], before[rest])


def test_8_bit_m_with_a_large_beta1(cuda_device):
    """Above 0.9 every m is dithered: a million equal m between two codes have the right mean, a block's largest stays the largest code,
    other steps give other codes, and what is not finite is NaN and leaves its block alone."""
    dev = cuda_device
    n = 1 << 20
    p = [torch.zeros(n, device=dev)]
    for sign in (1.0, -1.0):
        g = torch.full((n,), 1.3 * sign, device=dev)
        g[::256] = 7.0 * sign
        state = AdamWState.zeros(p, bits=8)
        adamw_step(p, [g], state, lr=0.0, betas=(0.95, 0.999))
        m = state.moments(0)[0].double().reshape(-1, 256) * sign / 0.05
        step = 2.0 ** (math.floor(math.log2(1.3 / (7.0 / 448))) - 3) * 7.0 / 448
        assert m[:, 1:].unique().numel() == 2 and (m[:, 0] - 7.0).abs().max() < 7 * 8 * E32
        assert abs(m[:, 1:].mean().item() - 1.3) < 5 * step / 2 / math.sqrt(m[:, 1:].numel()) + step * 2.0 ** -17 + 1.3 * 8 * E32
    first = state.exp_avg.view(torch.uint8).clone()
    again = AdamWState.zeros(p, bits=8)
    adamw_step(p, [g], again, lr=0.0, betas=(0.95, 0.999))
    assert torch.equal(again.exp_avg.view(torch.uint8), first)
    again = AdamWState.zeros(p, bits=8)
    adamw_step(p, [g], again, lr=0.0, betas=(0.95, 0.999), step=2)
    assert not torch.equal(again.exp_avg.view(torch.uint8), first)
    bad = g.clone()
    bad[5], bad[300], bad[777] = math.nan, math.inf, -math.inf
    voided = torch.zeros(n, dtype=torch.bool, device=dev)
    voided[[5, 300, 777]] = True
    got = AdamWState.zeros(p, bits=8)
    adamw_step([p[0].clone()], [bad], got, lr=0.0, betas=(0.95, 0.999))
    m, v = got.moments(0)
    assert torch.isnan(m[voided]).all() and torch.isnan(v[voided]).all()
    assert torch.equal(got.exp_avg.view(torch.uint8)[~voided], first[~voided])


def test_8_bit_moments_follow_a_falling_gradient(cuda_device):
    """Gradients of one element fall to zero while its block's largest stays: rounding to nearest would hold its root for ever
    (a step changes it by 0.05 %, half a code's distance is 3 %); after 3000 steps with b2 = 0.999 it has shrunk to exp(-1.5)
    = 0.22 of itself, give or take the walk's deviation of some 25 %."""
    dev = cuda_device
    n = 256 * 64
    p, state = [torch.zeros(n, device=dev)], AdamWState.zeros([torch.zeros(n, device=dev)], bits=8)
    hot = torch.zeros(n, device=dev)
    hot[::256] = 4.0
    adamw_step(p, [torch.ones(n, device=dev) + hot], state, lr=0.0, betas=(0.9, 0.0))
    for _ in range(3000):
        adamw_step(p, [hot + (hot > 0)], state, lr=0.0, betas=(0.9, 0.999))
    roots = state.moments(0)[1].sqrt().reshape(-1, 256)[:, 1:]
    assert 0.17 < roots.double().square().mean().sqrt().item() < 0.3 and 0.17 < roots.mean().item() < 0.27


def test_what_is_not_finite_stays_by_itself(cuda_device):
    """8 bits: NaN, infinity and an overflowing square void their own element and no other of the block; 32 bits the same."""
    dev = cuda_device
    for bits in (8, 32):
        g = torch.randn(1000, generator=torch.Generator().manual_seed(3)).to(dev)
        clean = g.clone()
        g[5], g[300], g[301], g[302] = math.nan, math.inf, -math.inf, 1e25
        bad = torch.zeros(1000, dtype=torch.bool, device=dev)
        bad[[5, 300, 301, 302]] = True
        clean[bad] = 0.0
        got = []
        for t in (g, clean):
            p = [torch.ones(1000, device=dev)]
            state = AdamWState.zeros(p, bits=bits)
            adamw_step(p, [t], state, **RULE)
            adamw_step(p, [t.nan_to_num(0.0, 0.0, 0.0).clamp(-10, 10)], state, **RULE)
            got.append((p[0], *state.moments(0)))
        for a, b in zip(*got):
            assert torch.equal(a[~bad], b[~bad])
        assert torch.isnan(got[0][1][[5, 300, 301]]).logical_or(torch.isinf(got[0][1][[5, 300, 301]])).all()
        assert not torch.isfinite(got[0][2][bad]).any()


@pytest.mark.parametrize("bits", [32, 8])
def test_offsets_beyond_32_bits(cuda_device, bits):
    """A tensor of more than 2^31 elements and one behind it: the first step moves a weight by lr against its gradient's sign, whatever
    the gradient's size, at both ends; the rest stays."""
    dev = cuda_device
    n = (1 << 31) + 300
    params = [torch.zeros(n, dtype=torch.bfloat16, device=dev), torch.zeros(1000, dtype=torch.bfloat16, device=dev)]
    grads = [torch.zeros_like(p) for p in params]
    places = [0, 5, 1 << 30, n - 257, n - 1]
    for k, at in enumerate(places):
        grads[0][at] = 0.5 - k % 2
    grads[1][[0, 999]] = -1.0
    state = AdamWState.zeros(params, bits=bits)
    adamw_step(params, grads, state, lr=0.25, weight_decay=0.0)
    assert [params[0][at].item() for at in places] == [-0.25, 0.25, -0.25, 0.25, -0.25]
    assert torch.count_nonzero(params[0]).item() == len(places) and params[1].tolist() == [0.25] + [0.0] * 998 + [0.25]
    for k, at in enumerate(places):
        assert state.exp_avg.float()[at].item() * (0.5 - k % 2) > 0 if bits == 8 else state.exp_avg[at].item() == pytest.approx(0.1 * (0.5 - k % 2))


@pytest.mark.parametrize("bits", [32, 8])
def test_tensors_without_elements_alone(cuda_device, bits):
    """A group of one dtype may hold nothing else; they count their steps like any other.  The other group moves by half, of which 16 x 2^-24
    may be missing (as above) and 1e-8 to eps; 3 x 2^-24 of 1 for the parameter."""
    p = torch.nn.Parameter(torch.zeros(0, 5, dtype=torch.bfloat16, device=cuda_device))
    q = torch.nn.Parameter(torch.ones(3, device=cuda_device))
    opt = AdamW([p, q], lr=0.5, weight_decay=0.0, bits=bits, master=True)
    p.grad, q.grad = torch.zeros_like(p), torch.ones_like(q)
    opt.step()
    assert (q - 0.5).abs().max().item() <= 0.5 * (16 * E32 + 1e-8) + 3 * E32 and [s["step"] for s in opt.state_dict()["state"].values()] == [1, 1]


def test_tensors_that_share_memory_are_refused(cuda_device):
    dev = cuda_device
    p = torch.zeros(1000, device=dev)
    g = torch.zeros(1000, device=dev)
    for pair in ([p, p], [p[:600], p[400:]]):
        state = AdamWState.zeros(pair)
        with pytest.raises(OptimizerInputError, match="share memory"):
            adamw_step(pair, [g[:t.numel()] for t in pair], state, **RULE)
    touching = [p[:500], p[500:]]
    adamw_step(touching, [g[:500], g[500:]], AdamWState.zeros(touching), **RULE)


def test_tensors_of_different_ages_that_share_memory_are_refused(cuda_device):
    """A launch for each age must not get round the check, nor move some tensors before another one is refused."""
    dev = cuda_device
    p = torch.ones(1000, device=dev)
    g = [torch.ones(1000, device=dev), torch.ones(1000, device=dev)]
    for pair, grads in (([p, p], g), ([p[:600], p[400:]], [g[0][:600], g[1][:600]]), ([p, torch.ones(1000, device=dev)], [g[0], p])):
        state = AdamWState.zeros(pair)
        state.steps = [0, 4]
        with pytest.raises(OptimizerInputError, match="share memory"):
            adamw_step(pair, grads, state, **RULE)
        assert (p == 1).all() and state.steps == [0, 4] and (state.exp_avg == 0).all()


def test_refusals(cuda_device):
    dev = cuda_device
    p, g = [torch.zeros(8, 4, device=dev)], [torch.zeros(8, 4, device=dev)]
    s = AdamWState.zeros(p)
    s8 = AdamWState.zeros(p, bits=8)
    m32 = torch.zeros(256, device=dev)
    bad = [
        lambda: adamw_step(p, g + g, s, lr=0.1), lambda: adamw_step(p, [g[0].cpu()], s, lr=0.1), lambda: adamw_step(p, [g[0].half()], s, lr=0.1),
        lambda: adamw_step(p, [g[0][:4]], s, lr=0.1), lambda: adamw_step([p[0].t()], g, s, lr=0.1), lambda: adamw_step([p[0].double()], g, s, lr=0.1),
        lambda: adamw_step([p[0].cpu()], g, s, lr=0.1), lambda: adamw_step(p, g, s, lr=-0.1), lambda: adamw_step(p, g, s, lr=0.1, betas=(1.0, 0.9)),
        lambda: adamw_step(p, g, s, lr=0.1, betas=(0.9, -0.1)), lambda: adamw_step(p, g, s, lr=0.1, eps=-1.0), lambda: adamw_step(p, g, s, lr=0.1, weight_decay=-1.0),
        lambda: adamw_step(p, g, s, lr=0.1, step=0), lambda: adamw_step(p, [None], s, lr=0.1, out=(p, s)), lambda: adamw_step(p, g, s, lr=0.1, out=(p, s8)),
        lambda: adamw_step(p, g, s, lr=0.1, grad_scale=torch.ones(2, device=dev)), lambda: adamw_step(p, g, s, lr=0.1, grad_scale=torch.ones(1)),
        lambda: adamw_step(p, [g[0].to_sparse()], s, lr=0.1), lambda: adamw_step(p, g, s, lr=float("nan")),
        lambda: AdamWState.zeros(p, bits=16), lambda: AdamWState.zeros([]), lambda: AdamWState.zeros([p[0].cpu()]),
        lambda: AdamWState([32], m32[:128], m32), lambda: AdamWState([32], m32, m32.cpu()), lambda: AdamWState([32], m32, m32, scales=torch.zeros(1, 2, device=dev)),
        lambda: AdamWState([32], m32, m32, steps=[1, 2]), lambda: adamw_step(p, g, AdamWState.zeros(p, master=True), lr=0.1),
        lambda: adamw_step(p, g, AdamWState([32], torch.zeros(260, device=dev)[1:257], m32), lr=0.1),
        lambda: AdamW(p, bits=4),
    ]
    for k, call in enumerate(bad):
        with pytest.raises(OptimizerInputError):
            call()
            pytest.fail(f"call {k} was not refused")
    assert s.steps == [0] and (p[0] == 0).all()


def _model(dev, dtype=torch.float32, seed=0):
    torch.manual_seed(seed)
    return torch.nn.Sequential(torch.nn.Linear(33, 70), torch.nn.Tanh(), torch.nn.Linear(70, 9)).to(dev).to(dtype)


def _train(model, opt, steps, seed=1, scheduler=None):
    g = torch.Generator().manual_seed(seed)
    p = next(model.parameters())
    for _ in range(steps):
        x = torch.randn(16, 33, generator=g).to(p.device).to(p.dtype)
        opt.zero_grad(set_to_none=True)
        model(x).float().square().mean().backward()
        opt.step()
        if scheduler is not None:
            scheduler.step()


def test_optimizer_against_torch(cuda_device):
    """Ten steps with two groups and a schedule beside torch's AdamW in fp64.  Each step is within 16 x 2^-24 of its length, but
    gradients feed back; 1e-5 of the largest weight is some hundred of those."""
    a, b = _model(cuda_device), _model(cuda_device, torch.float64)
    groups = lambda m: [{"params": m[0].parameters()}, {"params": m[2].parameters(), "lr": 3e-3, "weight_decay": 0.2}]
    ours, theirs = AdamW(groups(a), lr=1e-2), torch.optim.AdamW(groups(b), lr=1e-2)
    _train(a, ours, 10, scheduler=torch.optim.lr_scheduler.ExponentialLR(ours, 0.8))
    _train(b, theirs, 10, scheduler=torch.optim.lr_scheduler.ExponentialLR(theirs, 0.8))
    for p, q in zip(a.parameters(), b.parameters()):
        assert (p.double() - q).abs().max() < 1e-5 * q.abs().max()


@pytest.mark.parametrize("bits,master", [(32, False), (8, True)])
def test_saved_and_loaded_optimizer_goes_on_alike(cuda_device, bits, master):
    import io
    dtype = torch.bfloat16 if master else torch.float32
    a = _model(cuda_device, dtype)
    opt = AdamW(a.parameters(), lr=1e-2, bits=bits, master=master)
    _train(a, opt, 4)
    buffer = io.BytesIO()
    torch.save({"model": a.state_dict(), "opt": opt.state_dict()}, buffer)
    buffer.seek(0)
    saved = torch.load(buffer)
    b = _model(cuda_device, dtype, seed=5)
    b.load_state_dict(saved["model"])
    other = AdamW(b.parameters(), lr=1.0, bits=bits, master=master)
    other.load_state_dict(saved["opt"])
    third, c = copy.deepcopy((opt, a))                            # one deep copy of both: the copy's groups hold the copied parameters
    for m, o in ((a, opt), (b, other), (c, third)):
        _train(m, o, 3, seed=2)
    for p, q, r in zip(a.parameters(), b.parameters(), c.parameters()):
        assert torch.equal(p, q) and torch.equal(p, r)
    one, two = opt.state_dict(), other.state_dict()
    assert one["param_groups"] == two["param_groups"] and all(s["step"] == 7 for s in one["state"].values())
    for k in one["state"]:
        for name, t in one["state"][k].items():
            if name != "step":
                assert torch.equal(t.view(torch.uint8), two["state"][k][name].view(torch.uint8))
    with pytest.raises(OptimizerInputError):
        AdamW(b.parameters(), bits=40 - bits, master=master).load_state_dict(saved["opt"])


@pytest.mark.parametrize("bits,master", [(32, False), (8, True)])
def test_a_refused_load_changes_nothing(cuda_device, bits, master):
    """Saved states that do not fit, the last parameter's alone among them: refused, and training goes on bit for bit as without them."""
    dtype = torch.bfloat16 if master else torch.float32
    a = _model(cuda_device, dtype)
    groups = [{"params": a[0].parameters()}, {"params": a[2].parameters(), "lr": 3e-3}]
    opt = AdamW(groups, lr=1e-2, bits=bits, master=master)
    _train(a, opt, 3)
    b, twin = copy.deepcopy((a, opt))
    good = copy.deepcopy(opt.state_dict())
    good["param_groups"][0]["lr"] = 7.0
    last = max(good["state"])
    for spoil in (lambda d: d["state"][last].pop("exp_avg_sq"), lambda d: d["state"][last].update(more=torch.zeros(1)),
                  lambda d: d["state"][last].update(exp_avg=d["state"][0]["exp_avg"]), lambda d: d["state"][last].update(step=-1),
                  lambda d: d["state"][last].update(exp_avg=d["state"][last]["exp_avg"].to(torch.float16)),
                  lambda d: d["state"].update({k: {**v, "exp_avg": v["exp_avg"].double()} for k, v in d["state"].items()}),
                  lambda d: d["param_groups"].pop(), lambda d: d["param_groups"][1]["params"].pop()):
        bad = copy.deepcopy(good)
        spoil(bad)
        with pytest.raises((OptimizerInputError, ValueError)):
            opt.load_state_dict(bad)
        assert opt.param_groups[0]["lr"] == 1e-2
    for m, o in ((a, opt), (b, twin)):
        _train(m, o, 2, seed=3)
    assert all(torch.equal(p, q) for p, q in zip(a.parameters(), b.parameters()))
    one, two = opt.state_dict(), twin.state_dict()
    assert all(s["step"] == 5 for s in one["state"].values())
    assert all(torch.equal(one["state"][k][n].view(torch.uint8), two["state"][k][n].view(torch.uint8))
               for k in one["state"] for n in one["state"][k] if n != "step")
    opt.load_state_dict(good)                                     # and the one that fits still loads
    assert opt.param_groups[0]["lr"] == 7.0 and all(s["step"] == 3 for s in opt.state_dict()["state"].values())


def test_mixed_dtypes_missing_gradients_and_versions(cuda_device):
    dev = cuda_device
    p = [torch.nn.Parameter(t) for t in (torch.ones(10, device=dev), torch.ones(300, device=dev, dtype=torch.bfloat16), torch.ones(7, device=dev))]
    opt = AdamW(p, lr=0.5, weight_decay=0.0, master=True)
    opt.step()                                                    # nothing to do
    p[0].grad, p[1].grad = torch.ones_like(p[0]), -torch.ones_like(p[1])
    y = (p[0] * p[0]).sum()                                       # keeps p[0] for its backward
    version = p[0]._version
    opt.step()
    assert (p[0] == 0.5).all() and (p[1] == 1.5).all() and (p[2] == 1.0).all() and p[0]._version > version
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()


def test_capture_is_refused_and_other_streams_work(cuda_device):
    dev = cuda_device
    p = torch.nn.Parameter(torch.ones(5000, device=dev))
    opt = AdamW([p], lr=0.5, weight_decay=0.0)
    p.grad = torch.ones_like(p)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        opt.step()
    torch.cuda.current_stream().wait_stream(side)
    assert (p == 0.5).all()
    refused, graph, one = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph(), torch.ones(1, device=dev)
    with pytest.raises(OptimizerInputError, match="captured"):
        with torch.cuda.graph(refused):
            one.add_(1)
            opt.step()
    torch.cuda.synchronize()
    # the step on lists with its number given can be captured; a replay repeats that very step
    state = AdamWState.zeros([p])
    to, after = [torch.empty_like(p)], AdamWState.zeros([p])
    with torch.cuda.graph(graph):
        adamw_step([p.detach()], [p.grad], state, lr=0.25, weight_decay=0.0, step=1, out=(to, after))
    for g in (1.0, -1.0):
        p.grad.fill_(g)
        graph.replay()
        torch.cuda.synchronize()
        assert (to[0] - (0.5 - 0.25 * g)).abs().max() < 1e-6
