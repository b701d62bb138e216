"""Cases that measure the operators of a language model's fine-tuning step: query and key norms with rotary
positions (``nc_ext_qk_norm_rope``), the clipped policy loss and the preference loss on logits
(``nc_ext_policy_loss``, ``nc_ext_preference_loss``) and AdamW with 8-bit states (``nc_ext_adamw8``).

With ``own`` false, ``run`` computes an operator in elementary torch operations; with ``own`` true it makes the calls
that a program makes of the framework, on tensors of the framework's own context. ``exact`` gives the same results from
the definitions in 64 bits, by other means than the plain form (complex rotations, automatic differentiation).
"""

import ctypes
import math

import numpy as np
import torch

own = False

DEV = "cuda"
INTERLEAVED, AXIS_FREQ = 1, 2  # NC_EXT_ROPE_* flags
BLOCK = 256                    # elements per 8-bit state block


# ---- cases ----------------------------------------------------------------------------------------


def listed():
    return [
        # one decoding step of 16 sequences, far into their contexts: the smallest call
        dict(name="rope_token", op="rope", batch=16, tokens=1, q_heads=8, k_heads=4, dim=64, sections="32", flags=0,
             far=500000, train=False),
        # the layer of the character-level transformer (64 x 128 tokens, 8 heads of 32) in training
        dict(name="rope_char_train", op="rope", batch=64, tokens=128, q_heads=8, k_heads=8, dim=32, sections="16",
             flags=0, far=0, train=True),
        # image patches (37 x 37), two axes, neighbouring pairs, a head size that is no power of two: an encoder's pass
        dict(name="rope_image", op="rope", batch=24, tokens=1369, q_heads=12, k_heads=12, dim=72, sections="18,18",
             flags=INTERLEAVED | AXIS_FREQ, far=0, train=False),
        # video tokens (time, height, width) with shared key heads in training: the largest
        dict(name="rope_video_train", op="rope", batch=4, tokens=4680, q_heads=16, k_heads=8, dim=128,
             sections="16,24,24", flags=0, far=0, train=True),
        # the character-level model tuned on rewards
        dict(name="policy_char", op="policy", batch=64, tokens=128, vocab=96, banned=0, kl=0.05, train=True),
        # scoring a few sampled sequences over a large vocabulary, no gradient
        dict(name="policy_score", op="policy", batch=4, tokens=61, vocab=128000, banned=17, kl=0.02, train=False),
        # a training batch over a vocabulary whose rows are not aligned: the largest
        dict(name="policy_train", op="policy", batch=4, tokens=2048, vocab=50001, banned=0, kl=0.05, train=True),
        # a few pairs of short answers
        dict(name="pref_small", op="pref", pairs=3, tokens=77, vocab=1000, smoothing=0.0, train=True),
        # pairs of answers of up to 700 tokens over an ordinary vocabulary
        dict(name="pref_train", op="pref", pairs=4, tokens=700, vocab=32000, smoothing=0.1, train=True),
        # the parameters of the small CNN
        dict(name="adamw8_cnn", op="adamw8", shapes="16x1x3x3,16,10x3136,10", decay=0.01),
        # embedding, one encoder layer and head of the character-level transformer
        dict(name="adamw8_char", op="adamw8", decay=0.01,
             shapes="256x96,256,768x256,768,256x256,256,1024x256,1024,256x1024,256,256,256,256,256,96x256,96"),
        # a few large matrices and vectors with odd ends
        dict(name="adamw8_large", op="adamw8", decay=0.1, shapes="8192x4096,4096x8192,4096x4096,50001x1024,4097,8191"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["rope", "policy", "pref", "adamw8"])
    if op == "rope":
        dim = 2 * rng.choice([8, 16, 20, 24, 32, 33, 36, 40, 48, 50, 64, 64, 96, 128])
        axes = rng.choice([1, 1, 2, 3])
        half = dim // 2
        cut = sorted(rng.randint(0, half) for _ in range(axes - 1))
        whole = half if rng.random() < 0.7 else rng.randint(max(1, half // 2), half)
        ends = [min(c, whole) for c in cut] + [whole]
        sections = ",".join(str(b - a) for a, b in zip([0] + ends[:-1], ends))
        kh = rng.choice([1, 2, 4, 7, 8, 12])
        qh = kh * rng.choice([1, 1, 2, 4])
        room = 4 * 4680 * 24 * 128 // (dim * (qh + kh))
        n = _log(rng, 1, room)
        batch = min(n, _log(rng, 1, 64))
        return dict(op="rope", batch=batch, tokens=max(1, n // batch), q_heads=qh, k_heads=kh, dim=dim,
                    sections=sections, flags=rng.choice([0, 1, 2, 3]), far=rng.choice([0, 0, 100000, 2000000]),
                    train=rng.random() < 0.6)
    if op in ("policy", "pref"):
        vocab = _log(rng, 2, 160000)
        room = (4 * 2048 * 50001 if op == "policy" else 8 * 700 * 32000) // vocab
        n = _log(rng, 2, min(room, 200000))
        if op == "policy":
            batch = min(n, _log(rng, 1, 64))
            return dict(op="policy", batch=batch, tokens=max(1, n // batch), vocab=vocab,
                        banned=rng.choice([0, 0, vocab // 3]), kl=rng.choice([0.0, 0.02, 0.1]),
                        train=rng.random() < 0.7)
        pairs = max(1, min(n // 2, _log(rng, 1, 32)))
        return dict(op="pref", pairs=pairs, tokens=max(1, n // (2 * pairs)), vocab=vocab,
                    smoothing=rng.choice([0.0, 0.1]), train=rng.random() < 0.7)
    left = _log(rng, 300, 135000000)
    sizes = [max(1, int(left * rng.random() ** 2)) for _ in range(rng.randint(1, 18))]
    over = max(1.0, sum(sizes) / left)
    return dict(op="adamw8", decay=rng.choice([0.0, 0.01, 0.1]),
                shapes=",".join(str(max(1, int(s / over))) for s in sizes))


def work(case):
    if case["op"] == "rope":
        n = case["batch"] * case["tokens"] * (case["q_heads"] + case["k_heads"]) * case["dim"]
        return {"bytes": (20 if case["train"] else 8) * n, "flops": (24 if case["train"] else 8) * n}
    if case["op"] in ("policy", "pref"):
        n = (case["batch"] if case["op"] == "policy" else 2 * case["pairs"]) * case["tokens"] * case["vocab"]
        return {"bytes": (8 if case["train"] else 4) * n, "flops": (8 if case["train"] else 4) * n}
    n = sum(math.prod(s) for s in _shapes(case))
    # weight and gradient read, weight written, codes read and written, and the states' values written
    return {"bytes": 24 * n, "flops": 40 * n}


# ---- inputs ---------------------------------------------------------------------------------------


def _ints(text):
    return [int(s) for s in text.split(",")]


def _shapes(case):
    return [[int(d) for d in s.split("x")] for s in case["shapes"].split(",")]


def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return g


def _rope_inputs(case, seed):
    g = _gen(seed)
    b, t, h, d = case["batch"], case["tokens"], case["q_heads"] + case["k_heads"], case["dim"]
    axes = len(_ints(case["sections"]))
    # projections of a few times unit size, with some heads much larger than others
    x = torch.randn(b, t, h, d, device=DEV, generator=g) * (0.3 + 4 * torch.rand(h, 1, device=DEV, generator=g))
    wq, wk = (1 + 0.3 * torch.randn(d, device=DEV, generator=g) for _ in range(2))
    if axes == 1:  # running positions from each sequence's own start
        pos = torch.arange(t, device=DEV).expand(b, t).unsqueeze(-1)
    else:  # a grid: the fastest axis runs over about the axes-th root of the tokens
        side = max(1, round(t ** (1.0 / axes)))
        at = torch.arange(t, device=DEV)
        pos = torch.stack([(at // side ** (axes - 1 - a)) % (side if a else t + 1) for a in range(axes)], -1)
        pos = pos.expand(b, t, axes)
    pos = pos + (torch.randint(0, case["far"] + 1, (b, 1, 1), device=DEV, generator=g) if case["far"] else 0)
    dy = torch.randn(b, t, h, d, device=DEV, generator=g) if case["train"] else None
    return x, wq, wk, pos.to(torch.int32).contiguous(), dy


def _logits(case, g, rows):
    z = torch.randn(rows, case["vocab"], device=DEV, generator=g)
    z *= 1 + 2 * torch.rand(rows, 1, device=DEV, generator=g)
    lab = torch.randint(0, case["vocab"] - case.get("banned", 0), (rows,), device=DEV, generator=g)
    z[torch.arange(rows, device=DEV), lab] += 4  # sampled tokens are likely ones
    if case.get("banned"):
        z[:, case["vocab"] - case["banned"]:] = -math.inf  # tokens that sampling may not take
    return z, lab.to(torch.int32)


def _logp(z, lab):
    return z.gather(1, lab.long()[:, None])[:, 0].double() - torch.logsumexp(z, 1).double()


def _policy_inputs(case, seed):
    g = _gen(seed)
    b, t = case["batch"], case["tokens"]
    z, act = _logits(case, g, b * t)
    rand = lambda: torch.randn(b * t, device=DEV, generator=g, dtype=torch.float64)  # noqa: E731
    # the policy has moved a little since it sampled: log ratios of about 0.15, none within 1e-4 of a clip border,
    # where 32 and 64 bits may fall on different sides
    ratio = 0.15 * rand()
    for edge in (math.log1p(-0.2), math.log1p(0.28)):
        near = (ratio - edge).abs() < 1e-4
        ratio = torch.where(near, torch.full_like(ratio, edge + 5e-4), ratio)
    lp = _logp(z, act)
    old, ref = (lp - ratio).float(), (lp + 0.3 * rand()).float()
    adv = rand().float()
    ends = torch.randint(1, t + 1, (b, 1), device=DEV, generator=g)
    mask = (torch.arange(t, device=DEV)[None] < ends).to(torch.int32).reshape(-1)
    return z, act, old, ref, adv, mask


def _pref_inputs(case, seed):
    g = _gen(seed)
    s, t = 2 * case["pairs"], case["tokens"]
    z, lab = _logits(case, g, s * t)
    ends = torch.randint(max(1, t // 2), t + 1, (s, 1), device=DEV, generator=g)
    mask = (torch.arange(t, device=DEV)[None] < ends).to(torch.int32)
    ref = (_logp(z, lab).view(s, t) * mask).sum(1) + 3 * torch.randn(s, device=DEV, generator=g, dtype=torch.float64)
    return z.view(s, t, -1), lab.view(s, t), mask, ref.float()


def _adam_inputs(case, seed):
    """Weights, gradients and first states of all tensors in one padded buffer each (whole blocks), and the slices."""
    g = _gen(seed)
    sizes = [math.prod(s) for s in _shapes(case)]
    at, spans = 0, []
    for n in sizes:
        spans.append((at, n))
        at += (n + BLOCK - 1) // BLOCK * BLOCK
    live = torch.zeros(at, dtype=torch.bool, device=DEV)
    for a, n in spans:
        live[a:a + n] = True
    # gradients whose size differs from row to row, some of them zero, as embeddings of unseen tokens are
    scale = torch.exp(2 * torch.randn(at // BLOCK, 1, device=DEV, generator=g)) * 1e-3
    scale[torch.rand(at // BLOCK, 1, device=DEV, generator=g) < 0.02] = 0
    make = lambda: torch.randn(at // BLOCK, BLOCK, device=DEV, generator=g)  # noqa: E731
    grad = (make() * scale).view(-1) * live
    m = (make() * scale * 0.3).view(-1) * live
    v = ((make() * scale).square() * 0.5).view(-1) * live
    w = make().view(-1) * 0.05 * live
    return w, grad, m, v, spans


HYPER = dict(lr=float(np.float32(1e-3)), beta1=float(np.float32(0.9)), beta2=float(np.float32(0.999)),
             eps=float(np.float32(1e-8)), start=100)  # the states stand after `start` steps


def prepare(case, seed):
    if own:
        return _prepare_own(case, seed)
    s = {"case": case}
    if case["op"] == "rope":
        s["in"], s["plan"] = _rope_inputs(case, seed), _pair_axes(case)
    elif case["op"] == "policy":
        s["in"] = _policy_inputs(case, seed)
    elif case["op"] == "pref":
        s["in"] = _pref_inputs(case, seed)
    else:
        w, grad, m, v, spans = _adam_inputs(case, seed)
        s.update(w=w, grad=grad, m=_encode_m(m), v=_encode_v(v), step=HYPER["start"], spans=spans)
        s["shapes"] = _shapes(case)
    return s


# ---- plain forms ----------------------------------------------------------------------------------


def run(state):
    if own:
        return _run_own(state)
    return {"rope": _plain_rope, "policy": _plain_policy, "pref": _plain_pref,
            "adamw8": _plain_adamw8}[state["case"]["op"]](state)


def _pair_axes(case):
    """The axis and the frequency of each of the dim / 2 pairs; pairs behind the last section stand still."""
    half, sections = case["dim"] // 2, _ints(case["sections"])
    axis = torch.tensor([a for a, n in enumerate(sections) for _ in range(n)] + [0] * (half - sum(sections)))
    i = torch.arange(half, dtype=torch.float64)
    turns = torch.arange(half) < sum(sections)
    if case["flags"] & AXIS_FREQ:  # each axis runs through all frequencies
        first = torch.tensor([sum(sections[:a]) for a, n in enumerate(sections) for _ in range(n)] + [0] * (half - sum(sections)))
        width = torch.tensor([n for n in sections for _ in range(n)] + [1] * (half - sum(sections)))
        power = (i - first) / width
    else:
        power = i / half
    return axis.to(DEV), torch.where(turns, 10000.0 ** -power, 0.0).to(DEV)


def _split(u, flags):
    return (u[..., 0::2], u[..., 1::2]) if flags & INTERLEAVED else u.chunk(2, -1)


def _join(a, b, flags):
    return torch.stack((a, b), -1).flatten(-2) if flags & INTERLEAVED else torch.cat((a, b), -1)


def _plain_rope(state):
    case = state["case"]
    x, wq, wk, pos, dy = state["in"]
    flags, hq = case["flags"], case["q_heads"]
    w = torch.cat((wq.expand(hq, -1), wk.expand(case["k_heads"], -1)))
    axis, freq = state["plan"]
    angle = (pos[..., axis].double() * freq)[:, :, None]  # 32 bits lose the angles of far positions
    c, s = angle.cos().float(), angle.sin().float()
    r = torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-6)
    n = x * r
    a, b = _split(n * w, flags)
    y = _join(a * c - b * s, b * c + a * s, flags)
    if dy is None:
        return y
    a, b = _split(dy, flags)
    g = _join(a * c + b * s, b * c - a * s, flags)
    gn = g * n
    dw = gn.sum((0, 1))
    dx = r * (g * w - n * (gn * w).mean(-1, keepdim=True))
    return y, dx, dw[:hq].sum(0), dw[hq:].sum(0)


def _plain_rows(z, lab):
    top = z.max(1, keepdim=True).values
    e = torch.exp(z - top)
    total = e.sum(1, keepdim=True)
    z_lab = z.gather(1, lab.long()[:, None])
    return ((z_lab - top).double() - torch.log(total.double()))[:, 0], e, total  # 32 bits lose the ratios' last digits


def _plain_rows_grad(e, total, lab, coef):
    d = e * (-coef[:, None] / total)
    d.scatter_add_(1, lab.long()[:, None], coef[:, None])
    return d


def _plain_policy(state):
    case = state["case"]
    z, act, old, ref, adv, mask = state["in"]
    w = mask != 0
    lp, e, total = _plain_rows(z, act)
    ratio = torch.exp(lp - old.double())
    away = ref.double() - lp
    each = -torch.minimum(ratio * adv, ratio.clamp(1 - 0.2, 1 + 0.28) * adv)
    each = each + case["kl"] * (torch.exp(away) - away - 1)
    count = w.sum().clamp(min=1)
    loss = torch.where(w, each, 0).sum().div(count).float()
    if not case["train"]:
        return loss, torch.where(w, lp, 0).float()
    moves = torch.where(adv >= 0, ratio <= 1 + 0.28, ratio >= 1 - 0.2)
    coef = torch.where(moves, -adv * ratio, 0) + case["kl"] * (1 - torch.exp(away))
    return loss, torch.where(w, lp, 0).float(), _plain_rows_grad(e, total, act, (torch.where(w, coef, 0) / count).float())


def _plain_pref(state):
    case = state["case"]
    z, lab, mask, ref = state["in"]
    s, t, vocab = z.shape
    p = s // 2
    lp, e, total = _plain_rows(z.view(-1, vocab), lab.view(-1))
    seq = torch.where(mask != 0, lp.view(s, t), 0).sum(1)
    gap = seq - ref
    h = 0.1 * (gap[:p] - gap[p:])
    eps = case["smoothing"]
    soft = lambda v: v.clamp(min=0) + torch.log1p(torch.exp(-v.abs()))  # noqa: E731
    loss = ((1 - eps) * soft(-h) + eps * soft(h)).mean().float()
    if not case["train"]:
        return loss, seq.float()
    push = (0.1 / p) * (1 / (1 + torch.exp(-h)) - (1 - eps))
    coef = torch.cat((push, -push)).float()[:, None] * (mask != 0)
    return loss, seq.float(), _plain_rows_grad(e, total, lab.view(-1), coef.view(-1)).view_as(z)


_steps = {}  # what a share has to reach for each code: (j - 1/2) to the power 2 or 4


def _table(power, count):
    if power not in _steps:
        _steps[power] = torch.tensor([(j - 0.5) ** power for j in range(1, count)], dtype=torch.float32, device=DEV)
    return _steps[power]


_M_UNIT, _V_UNIT = float(np.float32(1.0 / 127 ** 2)), float(np.float32(1.0 / 255.0 ** 4))
_LEAST = 2.0 ** -94  # blocks whose largest value is below stand for zero


def _codes(a, unit, steps):
    """The largest value of each block and, for each element, how many of the steps its share reaches."""
    a = a.view(-1, BLOCK)
    top = a.max(1, keepdim=True).values
    top = torch.where(top < _LEAST, 0, top)
    share = a * torch.where(top > 0, unit / top, 0)
    return top, torch.bucketize(share, steps, right=True)


def _encode_m(m):
    top, c = _codes(m.abs(), 127.0 ** 2, _table(2, 128))
    return top, torch.where(m.view(-1, BLOCK) < 0, -c, c).to(torch.int8)


def _encode_v(v):
    top, c = _codes(v, 255.0 ** 4, _table(4, 256))
    return top, torch.where((v.view(-1, BLOCK) > 0) & (top > 0), c.clamp(min=1), 0).to(torch.uint8)


def _decode_m(s):
    top, c = s
    c = c.float()
    m = (top * _M_UNIT) * (c * c.abs())
    return torch.where(c.abs() == 127, torch.sign(c) * top, m).view(-1)


def _decode_v(s):
    top, c = s
    c = c.float()
    q = c * c
    return torch.where(c == 255, top, ((top * _V_UNIT) * q) * q).view(-1)


def _plain_adamw8(s):
    h, decay = HYPER, s["case"]["decay"]
    s["step"] += 1
    b1, b2 = h["beta1"], h["beta2"]
    up1, up2 = float(np.float32(1) - np.float32(b1)), float(np.float32(1) - np.float32(b2))
    g = s["grad"]
    m = b1 * _decode_m(s["m"]) + up1 * g
    v = b2 * _decode_v(s["v"]) + (up2 * g) * g
    s["m"], s["v"] = _encode_m(m), _encode_v(v)
    move = (m / (1 - b1 ** s["step"])) / (torch.sqrt(v / (1 - b2 ** s["step"])) + h["eps"])
    s["w"] = s["w"] * (1 - h["lr"] * decay) - h["lr"] * move
    pick = lambda flat: [flat[a:a + n].view(shape) for (a, n), shape in zip(s["spans"], s["shapes"])]  # noqa: E731
    return {"w": pick(s["w"]), "m": pick(_decode_m(s["m"])), "v": pick(_decode_v(s["v"]))}


# ---- 64-bit results -------------------------------------------------------------------------------


def exact(case, seed):
    return {"rope": _exact_rope, "policy": _exact_policy, "pref": _exact_pref, "adamw8": _exact_adamw8}[case["op"]](case, seed)


def _exact_rope(case, seed):
    x, wq, wk, pos, dy = (None if v is None else v.double() for v in _rope_inputs(case, seed))
    half, hq = case["dim"] // 2, case["q_heads"]
    for v in (x, wq, wk):
        v.requires_grad_(dy is not None)
    angle = torch.zeros(*pos.shape[:2], half, dtype=torch.float64, device=DEV)
    i = 0
    for axis, n in enumerate(_ints(case["sections"])):
        for j in range(n):
            power = j / n if case["flags"] & AXIS_FREQ else i / half
            angle[..., i] = pos[..., axis] * math.exp(-power * math.log(10000.0))
            i += 1
    turn = torch.polar(torch.ones_like(angle), angle)[:, :, None]
    unit = x / torch.sqrt((x * x).sum(-1, keepdim=True) / case["dim"] + 1e-6)
    u = torch.cat((unit[:, :, :hq] * wq, unit[:, :, hq:] * wk), 2)
    if case["flags"] & INTERLEAVED:
        y = torch.view_as_real(torch.view_as_complex(u.unflatten(-1, (half, 2))) * turn).flatten(-2)
    else:
        both = torch.complex(u[..., :half], u[..., half:]) * turn
        y = torch.cat((both.real, both.imag), -1)
    if dy is None:
        return y
    y.backward(dy)
    return y.detach(), x.grad, wq.grad, wk.grad


def _exact_policy(case, seed):
    z, act, old, ref, adv, mask = _policy_inputs(case, seed)
    z = z.double().requires_grad_(case["train"])
    keep = mask.nonzero()[:, 0]
    lp = torch.zeros(len(z), dtype=torch.float64, device=DEV)
    if len(keep):
        lp = lp.index_put((keep,), torch.distributions.Categorical(logits=z[keep], validate_args=False).log_prob(act[keep].long()))
    ratio = (lp - old.double())[keep].exp()
    a = adv.double()[keep]
    gain = torch.where(a >= 0, ratio.clamp(max=1.28), ratio.clamp(min=0.8)) * a
    away = (ref.double() - lp)[keep]
    loss = (case["kl"] * (torch.expm1(away) - away) - gain).sum() / max(1, len(keep))
    if not case["train"]:
        return loss, lp
    loss.backward()
    return loss.detach(), lp.detach(), z.grad


def _exact_pref(case, seed):
    z, lab, mask, ref = _pref_inputs(case, seed)
    z = z.double().requires_grad_(case["train"])
    lp = torch.log_softmax(z, -1).gather(-1, lab.long()[..., None])[..., 0]
    seq = (lp * mask).sum(1)
    won, lost = (seq - ref.double()).chunk(2)
    h = 0.1 * (won - lost)
    eps = case["smoothing"]
    log_sig = torch.nn.functional.logsigmoid
    loss = -((1 - eps) * log_sig(h) + eps * log_sig(-h)).mean()
    if not case["train"]:
        return loss, seq
    loss.backward()
    return loss.detach(), seq.detach(), z.grad


def _exact_adamw8(case, seed):
    """The weights after the step from the values that the first states' codes stand for; the new states have no value
    in 64 bits of their own, they are rounded to 8."""
    w, grad, m, v, spans = _adam_inputs(case, seed)
    h, t = HYPER, HYPER["start"] + 1
    m, v = _decode_m(_encode_m(m)).double(), _decode_v(_encode_v(v)).double()
    grad = grad.double()
    m = torch.lerp(grad, m, h["beta1"])
    v = torch.lerp(grad * grad, v, h["beta2"])
    rate = h["lr"] * math.sqrt(1 - h["beta2"] ** t) / (1 - h["beta1"] ** t)
    w = w.double() - h["lr"] * case["decay"] * w.double() - rate * m / (v.sqrt() + h["eps"] * math.sqrt(1 - h["beta2"] ** t))
    return {"w": [w[a:a + n].view(shape) for (a, n), shape in zip(spans, _shapes(case))], "m": [None] * len(spans),
            "v": [None] * len(spans)}


# ---- the framework's calls ------------------------------------------------------------------------

_engine = None


class _Engine:
    """The one context that a program has, and its tensors as torch sees them (the same device memory)."""

    def __init__(self):
        from newch_b200 import capi

        self.capi, self.L = capi, capi.load_b200()
        self.ctx = self.L.nc_init(ctypes.byref(capi.Config(0, 1, 0, 0)))
        self.check()

    def check(self):
        if not self.L.nc_ok(self.ctx):
            raise RuntimeError(self.L.nc_error(self.ctx).decode())

    def view(self, t, held=None, write=0):
        """t as torch sees it. Made once for a program's state; it keeps the state's memory from being given back."""
        p = self.L.nc_ext_device_data(t, write)
        if not p:
            self.check()
            raise RuntimeError("a tensor without device data")
        n, shape = self.L.nc_ndim(t), self.L.nc_shape(t)
        key = (p, tuple(shape[i] for i in range(n)), self.L.nc_get_dtype(t))
        views = held.views if held else {}
        if key not in views:
            kind = {self.capi.F32: "<f4", self.capi.I32: "<i4"}[key[2]]
            face = _Face()
            face.memory = held.memory if held else None
            face.__cuda_array_interface__ = dict(shape=key[1], typestr=kind, data=(p, False), version=2)
            views[key] = torch.as_tensor(face, device=DEV)
        return views[key]

    def tensor(self, x, grad=False):
        """A tensor of the framework's that outlives the step, with x's values."""
        dtype = self.capi.I32 if x.dtype == torch.int32 else self.capi.F32
        self.L.nc_persistent_begin(self.ctx)
        t = self.L.nc_empty(self.ctx, dtype, *self.capi.shape_arg(x.shape))
        self.L.nc_persistent_end(self.ctx)
        self.check()
        if x.numel():
            self.view(t, write=1).copy_(x)
        if grad:
            self.L.nc_set_requires_grad(t, 1)
        return t


class _Face:
    """Device memory as torch takes it, and whose it is."""


class _Memory:
    """A program's tensors and optimizer, given back when neither it nor a result of it is held any more."""

    def __init__(self):
        self.tensors, self.optim = [], None

    def __del__(self):
        L = _engine.L
        if self.optim:
            L.nc_optim_free(self.optim)
        for t in self.tensors:
            L.nc_release(t)


class _Held:
    """What a program has in hand."""

    def __init__(self, case):
        self.case, self.memory, self.views = case, _Memory(), {}


def _prepare_own(case, seed):
    global _engine
    if _engine is None:
        _engine = _Engine()
    e, s = _engine, _Held(case)
    L, capi = e.L, e.capi
    grad = bool(case.get("train"))
    hold = lambda x, g=False: s.memory.tensors.append(e.tensor(x, g)) or s.memory.tensors[-1]  # noqa: E731
    if case["op"] == "rope":
        x, wq, wk, pos, dy = _rope_inputs(case, seed)
        s.x, s.wq, s.wk, s.pos = hold(x, grad), hold(wq, grad), hold(wk, grad), hold(pos)
        s.dy = hold(dy) if grad else None
        sections = _ints(case["sections"])
        s.opts = capi.RopeOpts(case["q_heads"], len(sections), (ctypes.c_int * 3)(*sections), 10000.0, 1e-6, case["flags"])
    elif case["op"] == "policy":
        z, act, old, ref, adv, mask = _policy_inputs(case, seed)
        s.logits = hold(z, grad)
        s.rest = [hold(v) for v in (act, old, ref, adv, mask)]
        s.opts = capi.PolicyOpts(0.2, 0.28, case["kl"])
    elif case["op"] == "pref":
        z, lab, mask, ref = _pref_inputs(case, seed)
        s.logits = hold(z, grad)
        s.rest = [hold(v) for v in (lab, ref, mask)]
    else:
        w, g, m, v, spans = _adam_inputs(case, seed)
        shapes = _shapes(case)
        pick = lambda flat: [flat[a:a + n] for a, n in spans]  # noqa: E731
        s.params = [hold(x.view(shape), True) for x, shape in zip(pick(w), shapes)]
        o = capi.OptimOpts(HYPER["lr"], 0.0, case["decay"], HYPER["beta1"], HYPER["beta2"], HYPER["eps"])
        s.optim = s.memory.optim = L.nc_ext_adamw8(e.ctx, capi.ptr_array(s.params), len(s.params), o)
        e.check()
        for p, x, shape in zip(s.params, pick(g), shapes):
            dp = e.tensor(x.view(shape))
            torch.cuda.synchronize()
            L.nc_ext_backward_from(p, dp)
            L.nc_ext_synchronize(e.ctx)
            L.nc_release(dp)
        s.states = hold(torch.stack((torch.cat(pick(m)), torch.cat(pick(v)))))
        torch.cuda.synchronize()
        L.nc_ext_optim_put_state(s.optim, s.states)
        L.nc_optim_set_step(s.optim, HYPER["start"])
        L.nc_ext_synchronize(e.ctx)
        both, at = e.view(s.states, s, 1), 0
        s.out = {"w": [e.view(p, s) for p in s.params], "m": [], "v": []}
        for (_, n), shape in zip(spans, shapes):
            s.out["m"].append(both[0, at:at + n].view(shape))
            s.out["v"].append(both[1, at:at + n].view(shape))
            at += n
    torch.cuda.synchronize()
    e.check()
    return s


def _run_own(s):
    e, case = _engine, s.case
    L = e.L
    L.nc_step_end(e.ctx)  # the step before is over
    if case["op"] == "rope":
        if not case["train"]:
            return e.view(L.nc_ext_qk_norm_rope(s.x, s.wq, s.wk, s.pos, ctypes.byref(s.opts)), s)
        for t in (s.x, s.wq, s.wk):
            L.nc_clear_grad(t)
        y = L.nc_ext_qk_norm_rope(s.x, s.wq, s.wk, s.pos, ctypes.byref(s.opts))
        L.nc_ext_backward_from(y, s.dy)
        return e.view(y, s), *(e.view(L.nc_grad(t), s) for t in (s.x, s.wq, s.wk))
    if case["op"] == "adamw8":
        L.nc_optim_step(s.optim)
        L.nc_ext_optim_get_state(s.optim, s.states)
        return s.out
    more = ctypes.c_void_p()
    if case["train"]:
        L.nc_clear_grad(s.logits)
    if case["op"] == "policy":
        loss = L.nc_ext_policy_loss(s.logits, *s.rest, ctypes.byref(s.opts), ctypes.byref(more))
    else:
        loss = L.nc_ext_preference_loss(s.logits, *s.rest, 0.1, case["smoothing"], ctypes.byref(more))
    if not case["train"]:
        return e.view(loss, s), e.view(more.value, s)
    L.nc_backward(loss)
    return e.view(loss, s), e.view(more.value, s), e.view(L.nc_grad(s.logits), s)
