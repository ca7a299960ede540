"""Preference and policy losses against their definitions in 64 bits, and their refusals.

Tolerances count roundings (half a step: 2^-24 of an fp32 value, 2^-8 of a bf16 one).
Preference: log ratios and all that follows are formed in double, so a reward or the loss has one rounding and a gradient
three (the sequence's weight, its product with the upstream gradient, and the stored value): 4 x 2^-24 leaves one spare.
Policy: u = x - o is rounded once, which exp turns into |u| 2^-24, exp adds 2 ulps (4 x 2^-24), the product with A one rounding; the KL
term and its slope have at most 4 ulps of their own parts (expm1: 1 ulp = 2 x 2^-24; the series: 8 fused steps whose first term
dominates, then two products).  So a token's term is within (12 + |u|) 2^-24 of |A r| + c |kl| and its slope within as much of
|A r| + c |kl'|; weight, upstream and store add three roundings.
"""
import math

import pytest
import torch

from mlx_train_perf_b200 import LossInputError, policy_loss, preference_loss

pytestmark = pytest.mark.gpu

E32 = 2.0 ** -24
STORE = {torch.float32: E32, torch.bfloat16: 2.0 ** -8}


def _tokens(seqs, length, packed, dtype, seed, mask_kind="random"):
    g = torch.Generator().manual_seed(seed)
    shape = (seqs * length,) if packed else (seqs, length)
    x = -1.5 * torch.randn(shape, generator=g).abs()
    o, r = x + 0.15 * torch.randn(shape, generator=g), x + 0.4 * torch.randn(shape, generator=g)
    mask = torch.rand(shape, generator=g) < 0.6
    if mask_kind == "all":
        mask = None
    elif mask_kind == "row" and not packed:
        mask[0] = False                                           # a sequence without a token that counts
    cu = None
    if packed:
        cuts = torch.sort(torch.randint(0, seqs * length + 1, (seqs - 1,), generator=g)).values if length else torch.zeros(seqs - 1).long()
        if seqs > 2:
            cuts[1] = cuts[0]                                     # an empty sequence
        cu = torch.cat([torch.zeros(1).long(), cuts, torch.tensor([seqs * length])]).to(torch.int32)
    return x.to(dtype), o.to(dtype), r.to(dtype), mask, cu, g


def _ranges(x, cu):
    """For each sequence the indexes of its tokens in the flat batch."""
    if cu is None:
        s, n = x.shape
        return [range(i * n, (i + 1) * n) for i in range(s)]
    c = cu.tolist()
    return [range(a, b) for a, b in zip(c[:-1], c[1:])]


def _weights(mask, x):
    return torch.ones(x.numel(), dtype=torch.bool) if mask is None else mask.reshape(-1)


def _preference_ref(x, r, mask, cu, kind, beta, smoothing, margin, average, upstream=1.0, sign=1.0):
    w = _weights(mask, x)
    d = torch.where(w, sign * (x.reshape(-1).double() - (0 if r is None else r.reshape(-1).double())), 0.0)
    seqs = _ranges(x, cu)
    pairs = len(seqs) // 2
    counts = [max(1, int(w[list(s)].sum())) if average else 1 for s in seqs]
    l = [float(d[list(s)].sum()) / c for s, c in zip(seqs, counts)]
    loss, grad = 0.0, torch.zeros(x.numel(), dtype=torch.float64)
    for i in range(pairs):
        h = beta * (l[i] - l[pairs + i]) - margin
        if kind == "sigmoid":
            sp = lambda z: max(z, 0.0) + math.log1p(math.exp(-abs(z)))
            loss += (1 - smoothing) * sp(-h) + smoothing * sp(h)
            slope = smoothing - 1 / (1 + math.exp(h))
        elif kind == "hinge":
            loss += max(0.0, 1 - h)
            slope = -1.0 if h < 1 else 0.0
        else:
            loss += ((h - 0.5) / beta) ** 2
            slope = 2 * (h - 0.5) / beta ** 2
        for s, k in ((i, 1.0), (pairs + i, -1.0)):
            for t in seqs[s]:
                if w[t]:
                    grad[t] = sign * k * beta * slope / pairs / counts[s] * upstream
    return loss / pairs, torch.tensor([beta * v for v in l], dtype=torch.float64), grad.reshape(x.shape)


def _close(got, ref, tol, store=E32):
    """|got - ref| <= tol (absolute, elementwise or a number) plus the store's rounding of the value."""
    got, ref = got.detach().double().cpu(), torch.as_tensor(ref, dtype=torch.float64)
    worst = ((got - ref).abs() - tol - store * ref.abs()).max().item() if ref.numel() else 0.0
    assert not torch.isnan(got).any() and worst <= 0.0, worst


CASES = [(2, 1, False), (2, 1, True), (4, 33, False), (6, 257, True), (8, 5000, False), (2, 70001, True), (4, 2051, False), (3000, 3, False), (10, 0, False)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("seqs,length,packed", CASES)
@pytest.mark.parametrize("kind,average", [("sigmoid", False), ("hinge", True), ("squared", True)])
def test_preference(cuda_device, seqs, length, packed, kind, average, dtype):
    x, _, r, mask, cu, _ = _tokens(seqs, length, packed, dtype, 3, "row")
    dev = cuda_device
    smoothing = 0.1 if kind == "sigmoid" else 0.0
    leaf = x.to(dev).requires_grad_(True)
    out = preference_loss(leaf, r.to(dev), mask=mask.to(dev), cu_seqlens=None if cu is None else cu.to(dev), kind=kind, beta=0.2,
                          label_smoothing=smoothing, margin=0.03, average=average)
    (out.loss * 3.0).backward()
    loss, rewards, grad = _preference_ref(x, r, mask, cu, kind, 0.2, smoothing, 0.03, average, 3.0)
    _close(out.loss, loss, 1e-12)
    _close(torch.cat([out.chosen_rewards, out.rejected_rewards]), rewards, 1e-12)
    _close(leaf.grad, grad, 4 * E32 * grad.abs(), STORE[dtype])
    assert leaf.grad.dtype == dtype and not out.chosen_rewards.requires_grad


def test_preference_without_reference_and_from_losses(cuda_device):
    x, _, r, mask, _, _ = _tokens(4, 100, False, torch.float32, 5)
    dev = cuda_device
    out = preference_loss(x.to(dev), mask=mask.to(dev), beta=0.5)
    loss, rewards, _ = _preference_ref(x, None, mask, None, "sigmoid", 0.5, 0.0, 0.0, False)
    _close(out.loss, loss, 1e-12)
    nll = (-x).to(dev).requires_grad_(True)
    out = preference_loss(nll, (-r).to(dev), mask=mask.to(dev), beta=0.5, from_nll=True)
    loss, rewards, grad = _preference_ref(x, r, mask, None, "sigmoid", 0.5, 0.0, 0.0, False)
    out.loss.backward()
    _close(out.loss, loss, 1e-12)
    _close(out.chosen_rewards, rewards[:2], 1e-12)
    _close(nll.grad, -grad, 4 * E32 * grad.abs())


def test_preference_far_ratios_do_not_overflow(cuda_device):
    x = torch.zeros(2, 4, device=cuda_device)
    r = torch.tensor([[1e4] * 4, [-1e4] * 4], device=cuda_device)
    x.requires_grad_(True)
    out = preference_loss(x, r, beta=1.0)
    out.loss.backward()
    assert out.loss.item() == 8e4 and (x.grad[0] == -1).all() and (x.grad[1] == 1).all()


def _policy_ref(x, o, r, a, mask, cu, low, high, coef, kl_kind, normalize, upstream=1.0, sign=1.0):
    """loss, kl, share, gradient, and the bounds' scale of loss and gradient."""
    w = _weights(mask, x)
    seqs = _ranges(x, cu)
    x32, o32 = sign * x.reshape(-1).float(), sign * o.reshape(-1).float()
    if a.shape == x.shape:
        a = a.reshape(-1).double()
    else:
        per = torch.zeros(x.numel(), dtype=torch.float64)
        for s, t in enumerate(seqs):
            per[list(t)] = float(a[s, 0])
        a = per
    u32 = x32 - o32                                               # the comparison's own definition: in fp32
    clipped = ((a > 0) & (u32 > torch.tensor(math.log1p(high), dtype=torch.float32))) | \
              ((a < 0) & (u32 < torch.tensor(math.log1p(-low) if low < 1 else -math.inf, dtype=torch.float32)))
    u = x32.double() - o32.double()
    ratio = u.exp()
    gain = a * torch.where(clipped, torch.where(a > 0, 1.0 + high, 1.0 - low), ratio)
    slope = torch.where(clipped, 0.0, -a * ratio)
    if r is None:
        kl = kls = torch.zeros_like(u)
    else:
        z = sign * r.reshape(-1).double() - x32.double()
        kl, kls = {"k3": (torch.expm1(z) - z, -torch.expm1(z)), "k2": (z * z / 2, -z), "k1": (-z, torch.ones_like(z))}[kl_kind]
    term = -gain + coef * kl
    size = (12 + u.abs()) * E32 * (gain.abs() + coef * kl.abs())
    slope_size = (12 + u.abs()) * E32 * ((a * ratio).abs() * ~clipped + coef * kls.abs())
    n = max(1, int(w.sum()))
    weight = torch.zeros(x.numel(), dtype=torch.float64)
    for t in seqs:
        t = list(t)
        c = max(1, int(w[t].sum()))
        weight[t] = {"token": 1 / n, "sequence": 1 / (len(seqs) * c), "sum": 1.0}[normalize]
    inside = torch.zeros(x.numel(), dtype=torch.bool)
    for t in seqs:
        inside[list(t)] = True
    w = w & inside
    sel = lambda v: torch.where(w, v, 0.0)
    n = max(1, int(w.sum()))
    if normalize == "token":
        weight = inside / n
    return (sel(term * weight).sum(), sel(kl).sum() / n, sel(clipped.double()).sum() / n, sel((coef * kls + slope) * weight * upstream * sign).reshape(x.shape),
            sel(size * weight).sum(), sel(kl.abs()).sum() / n * 8 * E32, sel((slope_size + 3 * E32 * (coef * kls + slope).abs()) * weight * upstream).reshape(x.shape))


def _check_policy(out, leaf, ref, dtype):
    loss, kl, share, grad, t_loss, t_kl, t_grad = ref
    _close(out.loss, loss, t_loss)
    _close(out.kl, kl, t_kl)
    _close(out.clip_fraction, share, 0.0)
    _close(leaf.grad, grad, t_grad, STORE[dtype])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("seqs,length,packed", [c for c in CASES if c[0] != 10] + [(1, 9001, False), (5, 0, False)])
@pytest.mark.parametrize("normalize,kl,per_token", [("token", "k3", False), ("sequence", "k2", True), ("sum", "k1", True), ("sequence", None, False)])
def test_policy(cuda_device, seqs, length, packed, normalize, kl, per_token, dtype):
    x, o, r, mask, cu, g = _tokens(seqs, length, packed, dtype, 7, "row")
    a = torch.randn(x.shape if per_token else (seqs, 1), generator=g)
    dev = cuda_device
    leaf = x.to(dev).requires_grad_(True)
    coef = 0.0 if kl is None else 0.3
    out = policy_loss(leaf, o.to(dev), a.to(dev), ref_logps=None if kl is None else r.to(dev), mask=mask.to(dev),
                      cu_seqlens=None if cu is None else cu.to(dev), clip_low=0.1, clip_high=0.2, kl_coef=coef, kl=kl or "k3",
                      normalize=normalize)
    (out.loss * 2.0).backward()
    ref = _policy_ref(x, o, None if kl is None else r, a, mask, cu, 0.1, 0.2, coef, kl, normalize, 2.0)
    _check_policy(out, leaf, ref, dtype)


def test_policy_from_losses_and_mixed_types(cuda_device):
    x, o, r, mask, _, g = _tokens(4, 77, False, torch.float32, 9)
    a = torch.randn(4, 1, generator=g)
    dev = cuda_device
    o16 = o.to(torch.bfloat16)
    nll = (-x).to(dev).requires_grad_(True)
    out = policy_loss(nll, (-o16).to(dev), a.to(dev).bfloat16(), ref_logps=(-r).to(dev), mask=mask.to(dev), kl_coef=0.1, from_nll=True)
    out.loss.backward()
    ref = _policy_ref(-x, -o16.float(), -r, a.bfloat16().float(), mask, None, 0.2, 0.2, 0.1, "k3", "token", sign=-1.0)
    _check_policy(out, nll, ref, torch.float32)


def test_what_the_mask_leaves_out_does_not_matter(cuda_device):
    """Infinities, NaN and the types' lowest values at tokens that do not count change nothing, and get no gradient."""
    dev = cuda_device
    x, o, r, mask, _, g = _tokens(4, 301, False, torch.float32, 11)
    a = torch.randn(x.shape, generator=g)
    bad = torch.tensor([math.nan, math.inf, -math.inf, torch.finfo(torch.float32).min])[torch.randint(0, 4, x.shape, generator=g)]
    got = []
    for fill in (False, True):
        t = [torch.where(mask, v, bad) if fill else v for v in (x, o, r, a)]
        leaf, ol, rl, al = (v.to(dev) for v in t)
        leaf.requires_grad_(True)
        p = policy_loss(leaf, ol, al, ref_logps=rl, mask=mask.to(dev), kl_coef=0.1)
        q = preference_loss(leaf, rl, mask=mask.to(dev))
        (p.loss + q.loss).backward()
        got.append((p.loss, p.kl, p.clip_fraction, q.loss, q.chosen_rewards, leaf.grad))
    assert all(torch.equal(u, v) for u, v in zip(*got))
    assert (got[1][-1].cpu()[~mask] == 0).all()


def test_values_that_count_and_are_not_finite_are_seen(cuda_device):
    x = torch.zeros(2, 8, device=cuda_device)
    x[0, 3] = math.nan
    for kind in ("sigmoid", "hinge", "squared"):
        assert math.isnan(preference_loss(x, kind=kind).loss.item())
    a = torch.ones(2, 1, device=cuda_device)
    assert math.isnan(policy_loss(x, torch.zeros_like(x), a).loss.item())


def test_infinite_ratios_where_they_do_not_count(cuda_device):
    """A rejected sequence that the model rules out is a loss of zero, not NaN; a KL term that is only reported may be infinite."""
    x = torch.zeros(2, 4, device=cuda_device)
    x[1, 2] = -math.inf
    x.requires_grad_(True)
    out = preference_loss(x, beta=0.3)
    out.loss.backward()
    assert out.loss.item() == 0.0 and (x.grad == 0).all() and out.rejected_rewards.item() == -math.inf
    y = torch.zeros(2, 4, device=cuda_device, requires_grad=True)
    r = torch.zeros(2, 4, device=cuda_device)
    r[0, 1] = -math.inf
    a = torch.ones(2, 1, device=cuda_device)
    out = policy_loss(y, torch.zeros_like(r), a, ref_logps=r)
    out.loss.backward()
    assert out.loss.item() == -1.0 and out.kl.item() == math.inf and (y.grad == -0.125).all()


def test_strided_rows_and_empty_masks(cuda_device):
    """Rows of a wider tensor (the usual shift by one), columns of a transposed one, expanded references; nothing counts at all."""
    dev = cuda_device
    x, o, r, mask, _, g = _tokens(6, 129, False, torch.float32, 13)
    a = torch.randn(6, 1, generator=g)
    want = policy_loss(x[:, 1:].contiguous().to(dev), o[:, 1:].contiguous().to(dev), a.to(dev), ref_logps=r[:, 1:].contiguous().to(dev),
                       mask=mask[:, 1:].contiguous().to(dev), kl_coef=0.1)
    xs = x.to(dev).requires_grad_(True)
    got = policy_loss(xs[:, 1:], o.to(dev)[:, 1:], a.to(dev), ref_logps=r.t().contiguous().to(dev).t()[:, 1:], mask=mask.to(dev)[:, 1:], kl_coef=0.1)
    assert torch.equal(got.loss, want.loss) and torch.equal(got.kl, want.kl)
    got.loss.backward()
    assert (xs.grad[:, 0] == 0).all() and xs.grad[:, 1:].abs().sum() > 0
    one = r[:1].to(dev).expand(6, -1)
    assert torch.equal(preference_loss(x.to(dev), one).loss, preference_loss(x.to(dev), one.contiguous()).loss)
    leaf = x.to(dev).requires_grad_(True)
    none = torch.zeros_like(mask).to(dev)
    out = policy_loss(leaf, o.to(dev), a.to(dev), ref_logps=r.to(dev), mask=none, kl_coef=0.1)
    pref = preference_loss(leaf, r.to(dev), mask=none, average=True)
    (out.loss + pref.loss).backward()
    assert out.loss.item() == 0 and out.kl.item() == 0 and (leaf.grad == 0).all()
    assert abs(pref.loss.item() - math.log(2)) < 1e-7
    # a leaf that is broadcast to all rows gets the sum of their gradients
    row = x[0].to(dev).requires_grad_(True)
    full = x[0].to(dev).repeat(6, 1).requires_grad_(True)
    preference_loss(row.expand(6, -1), r.to(dev)).loss.backward()
    preference_loss(full, r.to(dev)).loss.backward()
    torch.testing.assert_close(row.grad, full.grad.sum(0), rtol=0, atol=6 * E32 * full.grad.abs().sum(0).max().item())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("offsets", [(0, 0, 0, 0), (1, 1, 1, 1), (3, 3, 3, 3), (0, 1, 0, 0), (2, 0, 0, 0), (0, 0, 0, 3), (0, 0, 2, 0)])
def test_arrays_that_begin_anywhere(cuda_device, offsets, dtype):
    """Rows of 3001 tokens whose arrays begin on and off a boundary of four tokens, alike and not: the gradients of contiguous copies,
    bit for bit, and their sums up to the order of additions in double."""
    dev = cuda_device
    g = torch.Generator().manual_seed(27)
    wide = lambda t, o: torch.cat([torch.zeros(4, o, dtype=t.dtype), t, torch.zeros(4, 8 - o, dtype=t.dtype)], 1).to(dev)[:, o:o + 3001]
    x, o, r, mask, _, _ = _tokens(4, 3001, False, dtype, 29)
    a = torch.randn(x.shape, generator=g)
    got = []
    for place in (lambda t, k: t.to(dev), lambda t, k: wide(t, offsets[k])):
        leaf = place(x, 0).detach().requires_grad_(True)
        ol, rl, ml, al = place(o, 1), place(r, 2), place(mask, 3), place(a, 2)
        p = policy_loss(leaf, ol, al, ref_logps=rl, mask=ml, kl_coef=0.2)
        q = preference_loss(leaf, rl, mask=ml, beta=0.01)
        got.append((p.loss, p.kl, q.loss, torch.autograd.grad(p.loss, leaf)[0], torch.autograd.grad(q.loss, leaf)[0]))
    for u, v in zip(got[0][:3], got[1][:3]):
        assert abs(u.item() - v.item()) <= 2 * E32 * abs(v.item()) + 1e-12
    assert torch.equal(got[0][3], got[1][3])
    assert (got[0][4] - got[1][4]).abs().max() <= 2 * STORE[dtype] * got[1][4].abs().max()   # its weight follows the sums


@pytest.mark.parametrize("index", [torch.int32, torch.int64])
def test_packed_tokens_outside_every_sequence(cuda_device, index):
    dev = cuda_device
    x, o, r, _, _, g = _tokens(1, 1000, True, torch.float32, 15)
    cu = torch.tensor([100, 400, 400, 777, 901], dtype=index, device=dev)
    a = torch.randn(4, 1, generator=g)
    leaf = x.to(dev).requires_grad_(True)
    out = policy_loss(leaf, o.to(dev), a.to(dev), ref_logps=r.to(dev), cu_seqlens=cu, kl_coef=0.2, normalize="sequence", validate_seqlens=True)
    out.loss.backward()
    _check_policy(out, leaf, _policy_ref(x, o, r, a, None, cu.cpu(), 0.2, 0.2, 0.2, "k3", "sequence"), torch.float32)
    assert (leaf.grad[:100] == 0).all() and (leaf.grad[901:] == 0).all()
    leaf.grad = None
    preference_loss(leaf, r.to(dev), cu_seqlens=cu).loss.backward()
    assert (leaf.grad[:100] == 0).all() and (leaf.grad[901:] == 0).all() and leaf.grad[100:901].ne(0).all()


def test_borders_out_of_range_stay_inside(cuda_device):
    """Borders beyond the batch are held at its ends: the same result as with the borders there."""
    dev = cuda_device
    x = _tokens(1, 500, True, torch.float32, 17)[0].to(dev)
    wild = torch.tensor([-50, 200, 10 ** 6], dtype=torch.int64, device=dev)
    tame = torch.tensor([0, 200, 500], dtype=torch.int64, device=dev)
    assert torch.equal(preference_loss(x, cu_seqlens=wild).loss, preference_loss(x, cu_seqlens=tame).loss)


def test_gradients_against_differences(cuda_device):
    """Central differences of the loss in 64-bit definitions are exact enough; here the kernels' own losses, moved by 2^-5 along one
    direction: the slope along it agrees to the second-order term (step^2 times third derivatives of order one) and rounding."""
    dev = cuda_device
    x, o, r, mask, _, g = _tokens(4, 50, False, torch.float32, 19)
    a, way = torch.randn(4, 1, generator=g).to(dev), torch.randn(x.shape, generator=g).to(dev) * 0.05
    step = 2.0 ** -5
    for f in (lambda t: preference_loss(t, r.to(dev), mask=mask.to(dev), beta=0.3).loss,
              lambda t: policy_loss(t, o.to(dev), a, ref_logps=r.to(dev), mask=mask.to(dev), clip_low=1.0, clip_high=1e6, kl_coef=0.5).loss):
        leaf = x.to(dev).requires_grad_(True)
        f(leaf).backward()
        slope = (leaf.grad.double() * way.double()).sum().item()
        got = (f(x.to(dev) + step * way).item() - f(x.to(dev) - step * way).item()) / (2 * step)
        assert abs(got - slope) < 2e-3 * abs(slope) + 2e-5, (got, slope)


def test_clipped_share_and_sides(cuda_device):
    """One token on each side of each bound, both signs of the advantage: which are clipped, and what they add."""
    dev = cuda_device
    u = torch.tensor([0.3, 0.1, -0.1, -0.3], device=dev).repeat(2, 1)
    a = torch.tensor([[1.0], [-1.0]], device=dev)
    x = u.clone().requires_grad_(True)
    out = policy_loss(x, torch.zeros_like(u), a, normalize="sum")
    out.loss.backward()
    assert (x.grad != 0).tolist() == [[False, True, True, True], [True, True, True, False]]
    assert out.clip_fraction.item() == 0.25
    want = -(1.2 + math.exp(0.1) + math.exp(-0.1) + math.exp(-0.3)) + (math.exp(0.3) + math.exp(0.1) + math.exp(-0.1) + 0.8)
    assert abs(out.loss.item() - want) < 16 * 12 * E32


def test_no_gradient_wanted_and_second_derivative(cuda_device):
    x, o, r, _, _, _ = _tokens(2, 64, False, torch.float32, 21)
    x, o, r = (t.to(cuda_device) for t in (x, o, r))
    a = torch.ones(2, 1, device=cuda_device)
    assert not policy_loss(x, o, a).loss.requires_grad
    leaf = x.clone().requires_grad_(True)
    with torch.no_grad():
        assert not policy_loss(leaf, o, a).loss.requires_grad and not preference_loss(leaf, r).loss.requires_grad
    loss = policy_loss(leaf, o, a).loss
    with pytest.raises(LossInputError, match="second derivative"):
        torch.autograd.grad(loss, leaf, create_graph=True)


def test_results_can_be_written_to(cuda_device):
    """`loss /= n` for accumulated batches, and statistics scaled in place: the gradient is that of the scaled loss."""
    x, o, r, _, _, _ = (t if t is None or not isinstance(t, torch.Tensor) else t.to(cuda_device) for t in _tokens(2, 64, False, torch.float32, 22))
    a = torch.ones(2, 1, device=cuda_device)
    for call in (lambda t: policy_loss(t, o, a, ref_logps=r, kl_coef=0.1), lambda t: preference_loss(t, r)):
        leaf = x.clone().requires_grad_(True)
        want, = torch.autograd.grad(call(leaf).loss * 0.25, leaf)
        out = call(leaf)
        loss = out.loss
        loss /= 4
        out[1].mul_(7.0)
        out[2].zero_()
        assert torch.equal(torch.autograd.grad(loss, leaf)[0], want)


def test_saved_tensors_moved_to_the_host_and_back(cuda_device):
    """Hooks that keep what the backward needs on the host: the gradient is formed from what comes back."""
    x, o, r, mask, _, _ = _tokens(4, 200, False, torch.float32, 23)
    dev = cuda_device
    a = torch.ones(4, 1, device=dev)
    got = []
    for hooks in (False, True):
        leaf = x.to(dev).requires_grad_(True)
        wide = mask.to(dev).repeat(1, 2)[:, :200]                 # a mask with a row stride
        with torch.autograd.graph.save_on_cpu() if hooks else torch.enable_grad():
            loss = policy_loss(leaf, o.to(dev), a, mask=wide).loss + preference_loss(leaf, r.to(dev), mask=wide).loss
        loss.backward()
        got.append(leaf.grad)
    assert torch.equal(*got)


def test_other_stream_and_captured(cuda_device):
    """Two calls on a side stream, and a captured forward and backward replayed on new inputs, against the eager calls."""
    dev = cuda_device
    x, o, r, mask, cu, g = _tokens(6, 700, True, torch.float32, 25)
    a = torch.randn(6, 1, generator=g).to(dev)
    x, o, r, mask, cu = (t.to(dev) for t in (x, o, r, mask, cu))

    def both(leaf):
        loss = policy_loss(leaf, o, a, ref_logps=r, mask=mask, cu_seqlens=cu, kl_coef=0.1).loss + preference_loss(leaf, r, mask=mask, cu_seqlens=cu).loss
        return loss, torch.autograd.grad(loss, leaf)[0]

    want = [both(t.clone().requires_grad_(True)) for t in (x, 0.5 * x)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        leaf = x.clone().requires_grad_(True)
        got = both(leaf)
        for _ in range(2):
            both(leaf)                                            # warm-up for the capture below
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got[0], want[0][0]) and torch.equal(got[1], want[0][1])
    del got
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = both(leaf)
    for k, t in enumerate((x, 0.5 * x)):
        with torch.no_grad():
            leaf.copy_(t)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out[0], want[k][0]) and torch.equal(out[1], want[k][1])


def test_offsets_beyond_32_bits(cuda_device):
    """More than 2^31 tokens, rows of up to 2^30 (the longest), and packed: every token's slope is the same, at the ends too."""
    dev = cuda_device
    for seqs, length in ((3, 1 << 30), (4, (1 << 29) + 5)):
        x = torch.zeros(seqs, length, dtype=torch.bfloat16, device=dev, requires_grad=True)
        a = torch.arange(1.0, seqs + 1, device=dev)[:, None]
        out = policy_loss(x, torch.zeros_like(x), a, normalize="sequence")
        grad, = torch.autograd.grad(out.loss, x)
        assert abs(out.loss.item() + a.mean().item()) <= 1e-6 * a.mean().item()
        want = (-a[:, 0].double() / (seqs * length))
        for at in (0, 1, length // 2, length - 1):
            assert ((grad[:, at].double() - want).abs() <= 2.0 ** -7 * want.abs()).all()
        del grad, out
    loss = preference_loss(x, beta=1.0)
    grad, = torch.autograd.grad(loss.loss, x)
    assert abs(loss.loss.item() - math.log(2)) < 1e-6
    assert (grad[:2, [0, length - 1]] == -0.25).all() and (grad[2:, [0, length - 1]] == 0.25).all()


def test_refusals(cuda_device):
    dev = cuda_device
    x = torch.zeros(4, 8, device=dev)
    a = torch.zeros(4, 1, device=dev)
    cu = torch.tensor([0, 4, 32], dtype=torch.int32, device=dev)
    flat = torch.zeros(32, device=dev)
    bad = [
        lambda: preference_loss(x[:3]), lambda: preference_loss(flat), lambda: preference_loss(x.half()),
        lambda: preference_loss(x, kind="other"), lambda: preference_loss(x, beta=0.0), lambda: preference_loss(x, label_smoothing=1.0),
        lambda: preference_loss(x, kind="hinge", label_smoothing=0.1), lambda: preference_loss(x, x[:, :4]),
        lambda: preference_loss(x, mask=torch.ones_like(x)), lambda: preference_loss(x, mask=torch.ones(4, 7, dtype=torch.bool, device=dev)),
        lambda: preference_loss(x, x.cpu()), lambda: preference_loss(x, cu_seqlens=cu), lambda: preference_loss(flat, cu_seqlens=cu.cpu()),
        lambda: preference_loss(flat, cu_seqlens=cu.float()), lambda: preference_loss(flat, cu_seqlens=cu[:1]),
        lambda: preference_loss(flat, cu_seqlens=torch.tensor([0, 9, 4], device=dev), validate_seqlens=True),
        lambda: preference_loss(flat, cu_seqlens=torch.tensor([0, 9, 33], device=dev), validate_seqlens=True),
        lambda: policy_loss(x, x, torch.zeros(4, device=dev)), lambda: policy_loss(x, x, a.cpu()), lambda: policy_loss(x, x, a.int()),
        lambda: policy_loss(x, x, a, kl_coef=0.1), lambda: policy_loss(x, x, a, clip_low=1.5), lambda: policy_loss(x, x, a, clip_high=-0.1),
        lambda: policy_loss(x, x, a, kl="k4"), lambda: policy_loss(x, x, a, normalize="mean"), lambda: policy_loss(x, x.half(), a),
        lambda: policy_loss(flat, flat, torch.zeros(3, 1, device=dev), cu_seqlens=cu), lambda: policy_loss(x[0, 0], x, a),
    ]
    for k, call in enumerate(bad):
        with pytest.raises(LossInputError):
            call()
            pytest.fail(f"call {k} was not refused")


def test_with_the_vocabulary_loss(cuda_device):
    """As a trainer runs them: per-token losses of the trained head's model and of a reference, then either objective; the gradient
    of the hidden states against the same chain in 64 bits.  Tolerance: the vocabulary loss's gradient, bf16, 1e-2 of its largest
    value (tests/test_ce_gpu.py), on losses that are within 2e-5 of theirs."""
    from mlx_train_perf_b200 import DenseHead, fused_linear_ce
    dev = cuda_device
    g = torch.Generator().manual_seed(31)
    s, n, d, v = 4, 60, 64, 500
    h = torch.randn(s, n, d, generator=g).to(torch.bfloat16)
    h_ref = (h.float() + 0.1 * torch.randn(s, n, d, generator=g)).to(torch.bfloat16)
    w = (torch.randn(v, d, generator=g) * d ** -0.5).to(torch.bfloat16)
    t = torch.randint(0, v, (s, n), generator=g)
    t[:, :9] = -100
    t[2, 40:] = -100
    mask = (t != -100).to(dev)
    a = torch.randn(s, 1, generator=g)
    head = DenseHead(w.to(dev), trainable=False)
    with torch.no_grad():
        ref = fused_linear_ce(h_ref.to(dev), head, t.to(dev))[0]

    def plain_nll(hidden):
        z = hidden.double() @ w.double().t()
        safe = t.clamp(min=0)
        return torch.where(t >= 0, z.logsumexp(-1) - z.gather(-1, safe[..., None])[..., 0], 0.0)

    plain_ref = plain_nll(h_ref)
    for which in ("policy", "preference"):
        leaf = h.to(dev).requires_grad_(True)
        nll = fused_linear_ce(leaf, head, t.to(dev))[0]
        if which == "policy":
            loss = policy_loss(nll, ref, a.to(dev), ref_logps=ref, mask=mask, kl_coef=0.1, from_nll=True).loss
        else:
            loss = preference_loss(nll, ref, mask=mask, from_nll=True).loss
        loss.backward()
        leaf64 = h.double().requires_grad_(True)
        x, r, w64 = -plain_nll(leaf64), -plain_ref, (t >= 0).double()
        if which == "policy":
            ratio = (x - r).exp()
            z = r - x
            f = -torch.minimum(ratio * a, ratio.clamp(0.8, 1.2) * a) + 0.1 * (torch.expm1(z) - z)
            want = (f * w64).sum() / w64.sum()
        else:
            l = ((x - r) * w64).sum(1)
            want = -torch.nn.functional.logsigmoid(0.1 * (l[:2] - l[2:])).mean()
        want.backward()
        assert abs(loss.item() - want.item()) < 5e-5 * max(1.0, abs(want.item()))
        assert (leaf.grad.double().cpu() - leaf64.grad).abs().max() <= 1e-2 * leaf64.grad.abs().max()


def test_forward_mode_derivatives_are_refused(cuda_device):
    """With and without a recorded gradient; beside a dual level a call without tangents gives what it gives outside."""
    from torch.autograd import forward_ad
    from mlx_train_perf_b200 import EmbeddingInputError, embedding_lookup
    x = torch.randn(4, 30, generator=torch.Generator().manual_seed(1)).to(cuda_device)
    a, ids = torch.ones(4, 1, device=cuda_device), torch.arange(4, device=cuda_device)
    want = preference_loss(x).loss, policy_loss(x, x + 0.1, a).loss, embedding_lookup(ids, x)
    for leaf in (x, x.clone().requires_grad_(True)):
        with forward_ad.dual_level():
            dual = forward_ad.make_dual(leaf, torch.ones_like(x))
            for call, error in ((lambda: preference_loss(dual), LossInputError), (lambda: policy_loss(dual, x, a), LossInputError),
                                (lambda: embedding_lookup(ids, dual), EmbeddingInputError)):
                with pytest.raises(error, match="forward-mode"):
                    call()
            got = preference_loss(x).loss, policy_loss(x, x + 0.1, a).loss, embedding_lookup(ids, x)
            assert all(torch.equal(p, q) for p, q in zip(got, want))


@pytest.mark.parametrize("length", [5, 4000])
def test_no_advantage_and_a_ratio_beyond_fp32(cuda_device, length):
    """exp(100) is infinite in fp32; times an advantage of zero it is still nothing, and other tokens' losses stay.  A NaN that counts is
    still one."""
    dev = cuda_device
    x = torch.zeros(2, length, device=dev, requires_grad=True)
    old = torch.tensor([[-100.0], [0.0]], device=dev).expand(2, length).contiguous()
    for a in (torch.tensor([[0.0], [1.0]], device=dev), torch.tensor([[-0.0], [1.0]], device=dev).expand(2, length).contiguous()):
        got = policy_loss(x, old, a)
        grad, = torch.autograd.grad(got.loss, x)
        assert got.loss.item() == -0.5 and got.clip_fraction.item() == 0.0
        assert (grad[0] == 0).all() and torch.allclose(grad[1], torch.full_like(grad[1], -0.5 / length), rtol=4 * E32, atol=0.0)
    old[0, 1] = math.nan
    assert torch.isnan(policy_loss(x, old, a).loss)


@pytest.mark.parametrize("length", [64, 5000])
def test_a_kl_term_beside_gains_that_cancel(cuda_device, length):
    """Tokens in pairs that differ in the sign of their advantage alone: what is left of the loss is the KL term, with its own roundings
    (4 x 2^-24 as above, half of it for the result) and none of the gains', which are 10^5 times larger."""
    dev = cuda_device
    g = torch.Generator().manual_seed(5)
    x = -torch.rand(2, length, generator=g).repeat_interleave(2, 1)
    old = x + 0.02 * torch.rand(2, length, generator=g).repeat_interleave(2, 1)
    ref = x + 0.03 * torch.randn(2, length, generator=g).repeat_interleave(2, 1)
    a = torch.randn(2, length, generator=g).repeat_interleave(2, 1) * torch.tensor([1.0, -1.0]).repeat(length)
    z = (ref - x).double()                                         # the kernel's own difference, rounded once
    want = (torch.expm1(z) - z).mean().item() * 0.04
    got = policy_loss(x.to(dev), old.to(dev), a.to(dev), ref_logps=ref.to(dev), kl_coef=0.04)
    assert want < 1e-4 and abs(got.loss.item() - want) <= 6 * E32 * want and abs(got.kl.item() * 0.04 - want) <= 6 * E32 * want
