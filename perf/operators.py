"""The steps of a fine-tuning run around the vocabulary loss and attention, as cases that can be timed and compared.

Four operators, each in a plain form and as the package's own call:

  pref    preference loss over pairs of sequences, from per-token log-probabilities under the trained and the
          reference model, and its gradient.
  policy  clipped policy loss with a KL term, from per-token log-probabilities under the trained, the sampling and the
          reference model and advantages, and its gradient.
  adamw   one AdamW step over a model's trained tensors, moments in 32 or in 8 bits, with or without fp32 masters.
  embed   scaled embedding lookup, and the gradient of the table.

Sizes: batches of 2 to 512 sequences of up to 8192 tokens; adapters of rank 8 to 64 on q / v projections, or all weights
of a small model; tables of 32 k to 152 k rows of 1024 to 4096 values, 1 to 16384 tokens.
"""
import itertools
import math

import torch

own = False

BLOCK = 256                      # elements that share a scale in 8-bit moments; tensors start at multiples of it
TOP = 448.0                      # largest e4m3 value
LR, BETAS, EPS, DECAY = 2e-4, (0.9, 0.999), 1e-8, 0.01


# ---------------------------------------------------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------------------------------------------------
def _objective(name, op, seqs, length, layout, dtype="fp32", **more):
    c = {"name": name, "op": op, "seqs": seqs, "length": length, "layout": layout, "dtype": dtype}
    c.update(more)
    return c


def _adamw(name, layers, hidden, bits, dtype, rank=0, vocab=0, master=False):
    return {"name": name, "op": "adamw", "layers": layers, "hidden": hidden, "rank": rank, "vocab": vocab, "bits": bits,
            "dtype": dtype, "master": master}


def _embed(name, tokens, dim, vocab, dtype="bf16", step="train", scale=1.0):
    return {"name": name, "op": "embed", "tokens": tokens, "dim": dim, "vocab": vocab, "dtype": dtype, "step": step,
            "scale": scale}


def listed():
    return [
        # two short pairs, one micro-batch of a small run: launches and host work
        _objective("pref_small", "pref", 4, 60, "padded", kind="sigmoid", average=False),
        # an ordinary batch of packed documents, odd total, log ratios averaged over the answer
        _objective("pref_packed", "pref", 32, 1333, "packed", kind="squared", average=True),
        # a full batch of long dialogues
        _objective("pref_long", "pref", 512, 4096, "padded", kind="sigmoid", average=False),
        # a group of sampled answers to one prompt, one micro-batch
        _objective("policy_small", "policy", 8, 61, "padded", normalize="token", per_token=False),
        # a batch of groups, packed, each sequence weighing the same
        _objective("policy_packed", "policy", 64, 1025, "packed", normalize="sequence", per_token=False),
        # a whole rollout batch, advantages per token
        _objective("policy_rollout", "policy", 512, 8192, "padded", normalize="token", per_token=True),
        # adapters of rank 8 on q / v of a 32-layer model: 128 small tensors
        _adamw("adamw_lora", 32, 4096, 32, "bf16", rank=8),
        # all weights of a small model in bf16 with fp32 masters and fp32 moments
        _adamw("adamw_full32", 8, 1024, 32, "bf16", vocab=32768, master=True),
        # all weights of a larger one, 8-bit moments
        _adamw("adamw_full8", 16, 2048, 8, "bf16", vocab=32768),
        # one short example on a small model
        _embed("embed_small", 60, 1024, 32768),
        # embeddings of a validation batch, scaled as some models do it, no gradient
        _embed("embed_eval", 2051, 4096, 151936, step="eval", scale=64.0),
        # a packed batch on the flagship model, trained table
        _embed("embed_train", 16384, 4096, 151936),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["pref", "policy", "adamw", "embed"])
    if op in ("pref", "policy"):
        length = _log_int(rng, 1, 8192)
        most = max(2, min(512, (512 * (4096 if op == "pref" else 8192)) // length))
        seqs = _log_int(rng, 2, most)
        layout, dtype = rng.choice(["padded", "packed"]), rng.choice(["fp32", "fp32", "bf16"])
        if op == "pref":
            c = _objective("", op, seqs + seqs % 2 if seqs < 512 else 512, length, layout, dtype,
                           kind=rng.choice(["sigmoid", "hinge", "squared"]), average=rng.random() < 0.5)
        else:
            c = _objective("", op, seqs, length, layout, dtype, normalize=rng.choice(["token", "sequence"]),
                           per_token=rng.random() < 0.5)
    elif op == "adamw":
        bits, dtype = rng.choice([8, 32]), rng.choice(["bf16", "fp32"])
        if rng.random() < 0.5:
            c = _adamw("", rng.randint(1, 32), 64 * rng.randint(4, 64) + rng.choice([0, 8, 13]), bits, dtype, rank=rng.choice([8, 16, 64]))
        else:
            c = _adamw("", rng.randint(1, 8), 64 * rng.randint(4, 20) + rng.choice([0, 1, 24]), bits, dtype, vocab=_log_int(rng, 1000, 32768),
                       master=dtype == "bf16" and rng.random() < 0.5)
    else:
        dtype = rng.choice(["bf16", "bf16", "fp32"])
        dim = 64 * rng.randint(4, 64) + rng.choice([0, 0, 8, 3])
        vocab = _log_int(rng, 1000, 151936)
        c = _embed("", _log_int(rng, 1, 16384), dim, vocab, dtype, rng.choice(["train", "train", "eval"]), rng.choice([1.0, math.sqrt(dim)]))
        if dtype == "fp32":
            c["vocab"] = min(vocab, 151936 // 2)
    del c["name"]
    return c


# ---------------------------------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------------------------------
def _shapes(c):
    """The trained tensors: A and B of q_proj / v_proj in every layer (4 query heads to a kv head), or a model's weights."""
    h, out = c["hidden"], []
    kv = max(1, h // 4)
    for _ in range(c["layers"]):
        if c["rank"]:
            out += [(c["rank"], h), (h, c["rank"]), (c["rank"], h), (kv, c["rank"])]
        else:
            out += [(h,), (h, h), (kv, h), (kv, h), (h, h), (h,), (11 * h // 4, h), (11 * h // 4, h), (h, 11 * h // 4)]
    return out + ([] if c["rank"] else [(c["vocab"], h), (h,)])


def _numel(shape):
    return math.prod(shape)


def _padded(n):
    return (n + BLOCK - 1) // BLOCK * BLOCK


def _total(c):
    return sum(_padded(_numel(s)) for s in _shapes(c))


def _dtype(c):
    return torch.bfloat16 if c["dtype"] == "bf16" else torch.float32


def _lengths(c, g):
    """`seqs` lengths that add up to the packed batch's size: random cuts, some sequences empty or of one token."""
    t = c["seqs"] * c["length"]
    cuts = torch.randint(0, t + 1, (c["seqs"] - 1,), generator=g)
    return torch.cat([torch.tensor([0]), torch.sort(cuts).values, torch.tensor([t])])


def _prepare_objective(c, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    s, n = c["seqs"], c["length"]
    shape = (s, n) if c["layout"] == "padded" else (s * n,)

    def normal(*size):
        return torch.randn(*size, generator=g, device="cuda")

    # log-probabilities of sampled tokens lie mostly between 0 and -5; an update moves them by tenths
    logps = -1.5 * normal(*shape).abs()
    near, far = logps + 0.1 * normal(*shape), logps + 0.3 * normal(*shape)
    state = {"case": c, "logps": logps.to(_dtype(c)), "old": near.to(_dtype(c)), "ref": far.to(_dtype(c)), "cu": None}
    state["logps"].requires_grad_(True)
    if c["layout"] == "packed":
        state["cu"] = _lengths(c, torch.Generator().manual_seed(seed)).to(torch.int32).cuda()
        state["mask"] = torch.rand(shape, generator=g, device="cuda") < 0.7
    else:
        # a prompt in front and padding behind carry no loss
        at = torch.arange(n, device="cuda")[None]
        first = torch.randint(0, n // 4 + 1, (s, 1), generator=g, device="cuda")
        last = torch.randint(n // 2, n + 1, (s, 1), generator=g, device="cuda")
        state["mask"] = (at >= first) & (at < last)
    if c["op"] == "policy":
        # rewards normalised within the batch, one for each answer, or each token's own
        state["advantages"] = normal(*shape) if c["per_token"] else normal(s, 1)
    return state


def _dither(n, step, device):
    """For each of n positions a number in [0, 2^20), fixed by the position and the step: 16 bits of a 32-bit mix of the
    position's pair and the step, and half a bit below them."""
    x = torch.arange((n + 1) // 2, device=device) + step * 0x3504F333
    x = (x * 0x1E3779B1) & 0xFFFFFFFF
    x = x ^ (x >> 16)
    x = (x * 0x7FEB352D) & 0xFFFFFFFF
    x = x ^ (x >> 15)
    x = (x * 0x046CA68B) & 0xFFFFFFFF
    x = x ^ (x >> 16)
    return torch.stack([x & 0xFFFF, x >> 16], dim=-1).reshape(-1)[:n] * 16 + 8


def _quantize(m, v, step):
    """Moments as e4m3 codes and a scale for each block of 256: m to the nearest code; sqrt(v) up or down by the
    position's dither, and never down to zero."""
    m, r = m.reshape(-1, BLOCK), v.sqrt().reshape(-1, BLOCK)
    sm, sr = m.abs().amax(1, keepdim=True) / TOP, r.amax(1, keepdim=True) / TOP
    m8 = torch.where(sm > 0, m / sm, 0.0).clamp(-TOP, TOP).to(torch.float8_e4m3fn)
    y = torch.where(sr > 0, r / sr, 0.0)
    d = _dither(y.numel(), step, y.device).to(torch.int32).reshape(y.shape)
    normal = (((y.view(torch.int32) + d) >> 20) << 20).view(torch.float32)
    small = torch.floor(y * 512 + d * 2.0 ** -20) / 512
    y8 = torch.where(y >= 2.0 ** -6, normal, small).clamp(max=TOP)
    y8 = torch.where(r > 0, y8.clamp(min=2.0 ** -9), 0.0).to(torch.float8_e4m3fn)
    return m8.reshape(-1), y8.reshape(-1), torch.cat([sm, sr], dim=1)


def _values(codes, scales, which):
    return (codes.float().reshape(-1, BLOCK) * scales[:, which:which + 1]).reshape(-1)


def _prepare_adamw(c, seed):
    """Parameters, gradients and moments of step 100, each kind in one buffer in which every tensor starts at a multiple
    of 256 elements; the buffers that take the results lie beside them."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    shapes = _shapes(c)
    n = _total(c)
    inside = torch.zeros(n, dtype=torch.bool, device="cuda")
    at = list(itertools.accumulate((_padded(_numel(s)) for s in shapes), initial=0))[:-1]
    for o, s in zip(at, shapes):
        inside[o:o + _numel(s)] = True

    def normal(scale):
        return (torch.randn(n, generator=g, device="cuda") * scale).masked_fill_(~inside, 0.0)

    # weights of a few hundredths; gradients of 1e-3, their size differing from block to block
    p = normal(0.02)
    size = torch.exp(torch.randn(n // BLOCK, 1, generator=g, device="cuda")).mul_(1e-3)
    grad = normal(1.0).reshape(-1, BLOCK).mul_(size).reshape(-1).to(_dtype(c))
    m = normal(0.3).reshape(-1, BLOCK).mul_(size).reshape(-1)
    v = normal(1.0).reshape(-1, BLOCK).mul_(size).reshape(-1).square_()
    state = {"case": c, "numels": [_numel(s) for s in shapes], "step": 101, "grad": grad}
    state["master"] = p if c["master"] else None
    state["p"] = p.to(_dtype(c))
    state["m"], state["v"], state["scales"] = (m, v, None) if c["bits"] == 32 else _quantize(m, v, 100)
    del m, v, size

    for k in ("p", "m", "v", "scales", "master"):
        state[k + "_out"] = None if state[k] is None else torch.zeros_like(state[k])

    def views(flat):
        return [flat[o:o + _numel(s)].view(s) for o, s in zip(at, shapes)]

    state["params"], state["grads"], state["params_out"] = views(state["p"]), views(state["grad"]), views(state["p_out"])
    return state


def _prepare_embed(c, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    n, d, v = c["tokens"], c["dim"], c["vocab"]
    weight = torch.randn(v, d, generator=g, device="cuda", dtype=_dtype(c))
    # words are used about as often as one over their rank; a tenth of the batch is padding
    u = torch.rand(n, generator=g, device="cuda", dtype=torch.float64)
    rank = torch.exp(u * math.log(v)).long() - 1
    ids = (rank * 7919 + 11) % v
    ids[n - n // 10:] = 0
    state = {"case": c, "ids": ids, "weight": weight.requires_grad_(c["step"] == "train")}
    if c["step"] == "train":
        state["d_out"] = torch.randn(n, d, generator=g, device="cuda", dtype=_dtype(c))
    return state


def prepare(case, seed):
    return {"pref": _prepare_objective, "policy": _prepare_objective, "adamw": _prepare_adamw, "embed": _prepare_embed}[case["op"]](case, seed)


# ---------------------------------------------------------------------------------------------------------------------
# plain forms
# ---------------------------------------------------------------------------------------------------------------------
BETA, SMOOTHING, MARGIN = 0.1, 0.1, 0.05
CLIP_LOW, CLIP_HIGH, KL = 0.2, 0.28, 0.04


def _sequence_of(state):
    """Each token's sequence, shaped like the tokens."""
    x, s = state["logps"], state["case"]["seqs"]
    if state["cu"] is None:
        return torch.arange(s, device=x.device)[:, None].expand(x.shape)
    return torch.searchsorted(state["cu"].long(), torch.arange(x.shape[0], device=x.device), right=True) - 1


def _sums(values, seq, s):
    return torch.zeros(s, dtype=torch.float64, device=values.device).index_add_(0, seq.reshape(-1), values.double().reshape(-1))


def _plain_pref(state):
    c, mask, s = state["case"], state["mask"], state["case"]["seqs"]
    x, r = state["logps"].detach(), state["ref"]
    seq = _sequence_of(state)
    length = _sums(mask, seq, s).clamp(min=1) if c["average"] else torch.ones(s, dtype=torch.float64, device=x.device)
    ratio = _sums(torch.where(mask, x.float() - r.float(), 0.0), seq, s) / length
    h = BETA * (ratio[:s // 2] - ratio[s // 2:]) - MARGIN
    if c["kind"] == "sigmoid":
        loss = (1 - SMOOTHING) * torch.log1p(torch.exp(-h)) + SMOOTHING * torch.log1p(torch.exp(h))
        slope = SMOOTHING - 1 / (1 + torch.exp(h))
    elif c["kind"] == "hinge":
        loss, slope = (1 - h).clamp(min=0), -(h < 1).double()
    else:
        off = h / BETA - 1 / (2 * BETA)
        loss, slope = off * off, 2 * off / BETA
    slope = BETA * slope / (s // 2)
    weight = (torch.cat([slope, -slope]) / length).float()
    grad = torch.where(mask, weight[seq], 0.0).to(x.dtype)
    rewards = (BETA * ratio).float()
    return {"loss": loss.mean().float(), "chosen": rewards[:s // 2], "rejected": rewards[s // 2:], "grad": grad}


def _plain_policy(state):
    c, mask, s = state["case"], state["mask"], state["case"]["seqs"]
    x, o, r = (state[k].detach().float() for k in ("logps", "old", "ref"))
    seq = _sequence_of(state)
    a = state["advantages"] if c["per_token"] else state["advantages"][:, 0][seq]
    u = x - o
    clipped = ((a > 0) & (u > math.log1p(CLIP_HIGH))) | ((a < 0) & (u < math.log1p(-CLIP_LOW)))
    bound = torch.where(a > 0, 1 + CLIP_HIGH, 1 - CLIP_LOW)
    ratio = torch.exp(u)
    z = (r - x).double()
    kl = torch.where(mask, torch.expm1(z) - z, 0.0)
    each = torch.where(mask, -a * torch.where(clipped, bound, ratio) + KL * kl, 0.0)
    slope = torch.where(clipped, 0.0, -a * ratio) - KL * torch.expm1(z).float()
    count = _sums(mask, seq, s)
    total = count.sum().clamp(min=1)
    if c["normalize"] == "token":
        loss, weight = each.sum() / total, (1 / total).expand(s)
    else:
        weight = 1 / (s * count.clamp(min=1))
        loss = (_sums(each, seq, s) * weight).sum()
    grad = torch.where(mask, slope * weight.float()[seq], 0.0).to(state["logps"].dtype)
    share = (clipped & mask).sum() / total
    return {"loss": loss.float(), "kl": (kl.sum() / total).float(), "clip": share.float(), "grad": grad}


def _plain_adamw(state):
    c, step = state["case"], state["step"]
    b1, b2 = BETAS
    g = state["grad"].float()
    p = (state["p"] if state["master"] is None else state["master"]).float()
    m, v = state["m"], state["v"]
    if c["bits"] == 8:
        m, v = _values(m, state["scales"], 0), _values(v, state["scales"], 1).square()
    m = b1 * m + (1 - b1) * g
    v = b2 * v + (1 - b2) * g * g
    root = v.sqrt() / math.sqrt(1 - b2 ** step) + EPS
    p = p * (1 - LR * DECAY) - LR / (1 - b1 ** step) * (m / root)
    out = {"p": p.to(_dtype(c))}
    if c["master"]:
        out["master"] = p
    if c["bits"] == 8:
        m, v, out["scales"] = _quantize(m, v, step)
    return {**out, "m": m, "v": v}


def _plain_embed(state):
    c, ids, w = state["case"], state["ids"], state["weight"].detach()
    out = {"out": (w[ids].float() * c["scale"]).to(w.dtype)}
    if c["step"] == "train":
        grad = torch.zeros(w.shape, dtype=torch.float32, device=w.device).index_add_(0, ids, state["d_out"].float())
        out["grad"] = (grad * c["scale"]).to(w.dtype)
    return out


# ---------------------------------------------------------------------------------------------------------------------
# the package's calls
# ---------------------------------------------------------------------------------------------------------------------
def _own_pref(state):
    from mlx_train_perf_b200 import preference_loss
    c = state["case"]
    got = preference_loss(state["logps"], state["ref"], mask=state["mask"], cu_seqlens=state["cu"], kind=c["kind"], beta=BETA,
                          label_smoothing=SMOOTHING if c["kind"] == "sigmoid" else 0.0, margin=MARGIN, average=c["average"])
    grad, = torch.autograd.grad(got.loss, state["logps"])
    return {"loss": got.loss.detach(), "chosen": got.chosen_rewards, "rejected": got.rejected_rewards, "grad": grad}


def _own_policy(state):
    from mlx_train_perf_b200 import policy_loss
    got = policy_loss(state["logps"], state["old"], state["advantages"], ref_logps=state["ref"], mask=state["mask"],
                      cu_seqlens=state["cu"], clip_low=CLIP_LOW, clip_high=CLIP_HIGH, kl_coef=KL, normalize=state["case"]["normalize"])
    grad, = torch.autograd.grad(got.loss, state["logps"])
    return {"loss": got.loss.detach(), "kl": got.kl, "clip": got.clip_fraction, "grad": grad}


def _own_adamw(state):
    from mlx_train_perf_b200 import AdamWState, adamw_step
    c = state["case"]
    now = AdamWState(state["numels"], state["m"], state["v"], scales=state["scales"], master=state["master"])
    after = AdamWState(state["numels"], state["m_out"], state["v_out"], scales=state["scales_out"], master=state["master_out"])
    adamw_step(state["params"], state["grads"], now, lr=LR, betas=BETAS, eps=EPS, weight_decay=DECAY, step=state["step"],
               out=(state["params_out"], after))
    out = {"p": state["p_out"], "m": state["m_out"], "v": state["v_out"]}
    if c["master"]:
        out["master"] = state["master_out"]
    if c["bits"] == 8:
        out["scales"] = state["scales_out"]
    return out


def _own_embed(state):
    from mlx_train_perf_b200 import embedding_lookup
    c = state["case"]
    with torch.set_grad_enabled(c["step"] == "train"):
        got = embedding_lookup(state["ids"], state["weight"], scale=c["scale"])
    out = {"out": got.detach()}
    if c["step"] == "train":
        out["grad"], = torch.autograd.grad(got, state["weight"], state["d_out"])
    return out


def run(state):
    op = state["case"]["op"]
    if own:
        return {"pref": _own_pref, "policy": _own_policy, "adamw": _own_adamw, "embed": _own_embed}[op](state)
    with torch.no_grad():
        return {"pref": _plain_pref, "policy": _plain_policy, "adamw": _plain_adamw, "embed": _plain_embed}[op](state)


def work(case):
    """Bytes: each input read once, each output written once.  Flops: a few operations a value."""
    c = case
    if c["op"] in ("pref", "policy"):
        t, item = c["seqs"] * c["length"], 2 if c["dtype"] == "bf16" else 4
        if c["op"] == "pref":
            return {"bytes": t * (3 * item + 1) + 4 * c["seqs"], "flops": 4.0 * t}
        return {"bytes": t * (4 * item + 1 + 4 * c["per_token"]) + 4 * c["seqs"], "flops": 20.0 * t}
    if c["op"] == "adamw":
        n, item = sum(_numel(s) for s in _shapes(c)), 2 if c["dtype"] == "bf16" else 4
        each = item + (8 + item if c["master"] else 2 * item) + (16 if c["bits"] == 32 else 4 + 16 / BLOCK)
        return {"bytes": n * each, "flops": 15.0 * n}
    n, d, v, item = c["tokens"], c["dim"], c["vocab"], 2 if c["dtype"] == "bf16" else 4
    moved = 8 * n + 2 * n * d * item
    if c["step"] == "train":
        moved += (n + v) * d * item
    return {"bytes": moved, "flops": 2.0 * n * d}


# ---------------------------------------------------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------------------------------------------------
def _exact_pieces(state):
    """Two functions: values of all tokens -> each sequence's sum (differences of the running sum at the sequences' borders), and
    a value of each sequence -> all its tokens."""
    s, x = state["case"]["seqs"], state["logps"]
    border = torch.arange(s + 1, device=x.device) * state["case"]["length"] if state["cu"] is None else state["cu"].long()

    def total(values):
        run_ = torch.cat([torch.zeros(1, dtype=torch.float64, device=x.device), values.reshape(-1).cumsum(0)])
        return run_[border[1:]] - run_[border[:-1]]

    def spread(per_sequence):
        return torch.repeat_interleave(per_sequence, border[1:] - border[:-1]).reshape(x.shape)

    return total, spread


def _exact_pref(state):
    c, s = state["case"], state["case"]["seqs"]
    half = s // 2
    w = state["mask"].double()
    total, spread = _exact_pieces(state)
    d = (state["logps"].detach().double() - state["ref"].double()) * w
    scale = 1 / total(w).clamp(min=1) if c["average"] else torch.ones(s, dtype=torch.float64, device=w.device)
    z = (total(d) * scale).requires_grad_(True)
    h = BETA * (z[:half] - z[half:]) - MARGIN
    if c["kind"] == "sigmoid":
        each = -(1 - SMOOTHING) * torch.nn.functional.logsigmoid(h) - SMOOTHING * torch.nn.functional.logsigmoid(-h)
    elif c["kind"] == "hinge":
        each = torch.relu(1 - h)
    else:
        each = (h / BETA - 0.5 / BETA) ** 2
    with torch.enable_grad():
        dz, = torch.autograd.grad(each.mean(), z)
    return {"loss": each.mean().detach(), "chosen": BETA * z[:half].detach(), "rejected": BETA * z[half:].detach(), "grad": spread(dz * scale) * w}


def _exact_policy(state):
    c, s = state["case"], state["case"]["seqs"]
    total, spread = _exact_pieces(state)
    w = state["mask"].double()
    x = state["logps"].detach().double().requires_grad_(True)
    a = state["advantages"].double()
    a = a if c["per_token"] else spread(a[:, 0])
    ratio = torch.exp(x - state["old"].double())
    free, held = ratio * a, ratio.clamp(1 - CLIP_LOW, 1 + CLIP_HIGH) * a
    gap = state["ref"].double() - x
    kl = torch.exp(gap) - gap - 1
    each = w * (-torch.minimum(free, held) + KL * kl)
    count = total(w)
    n = w.sum().clamp(min=1)
    loss = each.sum() / n if c["normalize"] == "token" else (each * spread(1 / count.clamp(min=1))).sum() / s
    grad, = torch.autograd.grad(loss, x)
    return {"loss": loss.detach(), "kl": ((w * kl).sum() / n).detach(), "clip": ((held < free).double() * w).sum() / n, "grad": grad}


def _spacing(y):
    """The distance between the e4m3 values around |y|."""
    e = torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6)))
    return torch.exp2(e - 3)


def _exact_adamw(state):
    c, t = state["case"], state["step"]
    if state["p"].numel() > 1_000_000_000:
        return None
    (b1, b2), f8 = BETAS, c["bits"] == 8
    rows = (lambda x: x.reshape(-1, BLOCK))
    p = (state["master"] if c["master"] else state["p"]).double()
    g = state["grad"].double()
    m, v = state["m"].double(), state["v"].double()
    if f8:
        sc = state["scales"].double()
        m, v = (rows(m) * sc[:, :1]).reshape(-1), (rows(v) * sc[:, 1:]).reshape(-1) ** 2
    m, v = torch.lerp(g, m, b1), torch.lerp(g ** 2, v, b2)
    p = p - LR * DECAY * p - LR * (m / (1 - b1 ** t)) / ((v / (1 - b2 ** t)) ** 0.5 + EPS)
    out = {"p": p, "m": m, "v": v}
    if c["master"]:
        out["master"] = p
    if f8:
        m, r = rows(m), rows(v ** 0.5)
        sc = torch.stack([m.abs().amax(1), r.amax(1)], dim=1) / TOP
        m, r = (torch.nan_to_num(x / k, nan=0.0) for x, k in ((m, sc[:, :1]), (r, sc[:, 1:])))
        up = _dither(r.numel(), t, r.device).double().reshape(r.shape) / 2 ** 20
        out["m"] = (torch.round(m / _spacing(m)) * _spacing(m)).clamp(-TOP, TOP).reshape(-1)
        coded = (torch.floor(r / _spacing(r) + up) * _spacing(r)).clamp(max=TOP)
        out["v"] = torch.where(r > 0, coded.clamp(min=2.0 ** -9), 0.0).reshape(-1)
        out["scales"] = sc
    return out


def _exact_embed(state):
    c, ids, w = state["case"], state["ids"], state["weight"].detach()
    out = {"out": w.index_select(0, ids).double() * c["scale"]}
    if c["step"] == "train":
        order = torch.argsort(ids, stable=True)
        rows, count = torch.unique_consecutive(ids[order], return_counts=True)
        sums = torch.segment_reduce(state["d_out"].double()[order], "sum", lengths=count, axis=0, unsafe=True)
        out["grad"] = torch.zeros(w.shape, dtype=torch.float64, device=w.device)
        out["grad"][rows] = sums * c["scale"]
    return out


def exact(case, seed):
    state = prepare(case, seed)
    return {"pref": _exact_pref, "policy": _exact_policy, "adamw": _exact_adamw, "embed": _exact_embed}[case["op"]](state)
