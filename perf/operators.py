"""The ordered and the random operators of the framework as a user's program calls them, with their plain forms.

Two operators, in the forms in which this framework meets them:

gated scan   h_t = a_t h_(t-1) + b_t along one axis, every channel on its own, with its gradients.  The compositing of depth-ordered
             layers is this recurrence (gate = 1 - alpha), and so are a decayed trace of per-Gaussian scores over an orbit and any
             gated recurrence over long sequences of channels.
draws        indices from softmax(logits / temperature), cut to the top k, the top p and the min p, by given random numbers:
             dense points of a scene (one row of N opacities, a million draws), serving (rows of a large alphabet, one draw each), a
             layer for every pixel (many short rows).

`own` False computes the plain forms with elementary torch operations, True calls the framework."""
import math

import numpy as np
import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


# ---------------------------------------------------------------------------------------------------------------- the cases
def listed():
    return [
        # one step of 64 streams of a recurrent layer while serving: nothing but latency
        dict(name="step serving bf16", op="step", B=64, D=2048, dtype="bf16", form="blend"),
        # a decayed trace of one score per Gaussian over the 60 views of the orbit, 1 M Gaussians
        dict(name="scan orbit trace f32", op="scan", B=1, T=60, D=1000000, dtype="f32", form="linear", train=False, ragged=False, reverse=False),
        # one long narrow sequence, odd length, forward only, with a carried-in state
        dict(name="scan long narrow f32", op="scan", B=1, T=100001, D=96, dtype="f32", form="linear", train=False, ragged=False, reverse=False),
        # long sequences in training: two of 32 k steps
        dict(name="train scan long bf16", op="scan", B=2, T=32768, D=512, dtype="bf16", form="linear", train=True, ragged=False, reverse=False),
        # an ordinary padded training batch, each sequence of its own length
        dict(name="train scan padded bf16", op="scan", B=8, T=2048, D=2048, dtype="bf16", form="blend", train=True, ragged=True, reverse=False),
        # 32 premultiplied RGBA layers of 800 x 800 over each other, with the gradients of colours, alphas and background
        dict(name="train layers 800x800 f32", op="layers", L=32, B=1, H=800, W=800, straight=False),
        # the smallest scene of the benchmark, one draw through all cuts: latency
        dict(name="draw one of 5000 f32", op="draw", R=1, V=5000, S=1, dtype="f32", dist="normal", temperature=0.7, top_k=50, top_p=0.9, min_p=0.02, rows=False),
        # a serving batch over a large alphabet, bf16 logits, every row with its own settings
        dict(name="draw serving bf16", op="draw", R=64, V=100003, S=1, dtype="bf16", dist="normal", temperature=0.8, top_k=200, top_p=0.95, min_p=0.01, rows=True),
        # a large batch cut by top p alone
        dict(name="draw batch top-p f32", op="draw", R=256, V=131072, S=1, dtype="f32", dist="normal", temperature=1.0, top_k=0, top_p=0.9, min_p=0.0, rows=False),
        # the dense points of a scene: a million draws from softmax(opacity) of 1 M Gaussians
        dict(name="draw points of 1M f32", op="draw", R=1, V=1000000, S=1000000, dtype="f32", dist="opacity", temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, rows=False),
        # the same for the largest scene, sharpened and without its faint splats
        dict(name="draw points of 6M top-p f32", op="draw", R=1, V=6000000, S=1000000, dtype="f32", dist="opacity", temperature=0.1, top_k=0, top_p=0.9, min_p=0.001, rows=False),
        # a layer for every pixel of an 800 x 800 image, four draws each; some pixels see no layer at all
        dict(name="draw layers 800x800 f32", op="draw", R=640000, V=32, S=4, dtype="f32", dist="layers", temperature=1.0, top_k=0, top_p=1.0, min_p=0.01, rows=False),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["step", "scan", "scan", "scan", "layers", "draw", "draw", "draw"])
    dtype = rng.choice(["f32", "bf16", "f16"])
    form = rng.choice(["linear", "blend", "over"])
    if op == "step":
        return dict(op=op, B=_log_int(rng, 1, 512), D=_log_int(rng, 256, 8192), dtype=dtype, form=form)
    if op == "scan":
        n = _log_int(rng, 1 << 14, 1 << (24 if dtype == "f32" else 25))       # steps x channels x sequences
        T = _log_int(rng, 1, min(100000, n // 16))
        B = _log_int(rng, 1, max(1, min(16, n // (16 * T))))
        return dict(op=op, B=B, T=T, D=max(1, n // (B * T)), dtype=dtype, form=form, train=rng.random() < 0.6, ragged=rng.random() < 0.4,
                    reverse=rng.random() < 0.3)
    if op == "layers":
        return dict(op=op, L=_log_int(rng, 1, 48), B=rng.choice([1, 1, 2]), H=_log_int(rng, 33, 600), W=_log_int(rng, 33, 600), straight=rng.random() < 0.5)
    kind = rng.choice(["rows", "points", "short"])
    cut = dict(temperature=round(rng.uniform(0.3, 1.5), 3), top_k=rng.choice([0, 0, _log_int(rng, 1, 2000)]), top_p=rng.choice([1.0, round(rng.uniform(0.1, 0.99), 3)]),
               min_p=rng.choice([0.0, round(rng.uniform(0.001, 0.2), 4)]))
    if kind == "rows":
        V = _log_int(rng, 1000, 260000)
        return dict(op="draw", R=_log_int(rng, 1, min(512, (1 << 24) // V)), V=V, S=rng.choice([1, 1, 1, _log_int(rng, 2, 64)]), dtype=dtype, dist="normal", rows=rng.random() < 0.5, **cut)
    if kind == "points":
        return dict(op="draw", R=1, V=_log_int(rng, 5000, 4000000), S=_log_int(rng, 1000, 1000000), dtype="f32", dist="opacity", rows=False, **cut)
    return dict(op="draw", R=_log_int(rng, 1000, 200000), V=_log_int(rng, 2, 300) if rng.random() < 0.5 else _log_int(rng, 2, 64), S=rng.choice([1, 1, _log_int(rng, 2, 16)]), dtype=dtype,
                dist="layers", rows=False, **cut)


# ---------------------------------------------------------------------------------------------------------------- the inputs
def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _normal(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def _uniform(g, *shape, dtype=torch.float32):
    return torch.rand(*shape, generator=g, device="cuda", dtype=dtype)


def _gate(g, form, *shape):
    """What a trained recurrence's gates look like: mostly remembering, here and there a reset.  `blend` and `over` gates are the share of the new input."""
    keep = torch.sigmoid(2.0 + 1.5 * _normal(g, *shape))
    return keep if form == "linear" else 1.0 - keep


def prepare(case, seed):
    g = _generator(seed)
    c = dict(case)
    op = c["op"]
    if op == "step":
        t = DTYPES[c["dtype"]]
        return dict(case=c, state=_normal(g, c["B"], c["D"]), gate=_gate(g, c["form"], c["B"], c["D"]).to(t), x=_normal(g, c["B"], c["D"]).to(t))
    if op == "scan":
        t = DTYPES[c["dtype"]]
        B, T, D, train = c["B"], c["T"], c["D"], c["train"]
        s = dict(case=c, gate=_gate(g, c["form"], B, T, D).to(t), x=_normal(g, B, T, D).to(t), initial=_normal(g, B, D), lengths=None)
        if c["ragged"]:
            s["lengths"] = torch.randint(0, T + 1, (B,), generator=g, device="cuda", dtype=torch.int32)
        if train:
            s["d_states"], s["d_last"] = _normal(g, B, T, D).to(t), _normal(g, B, D)
            for k in ("gate", "x", "initial"):
                s[k].requires_grad_(True)
        return s
    if op == "layers":
        L, B, H, W = c["L"], c["B"], c["H"], c["W"]
        alpha = _uniform(g, L, B, 1, H, W).square_()                   # splat layers: mostly thin
        rgb = _uniform(g, L, B, 3, H, W)
        if not c["straight"]:
            rgb.mul_(alpha)
        s = dict(case=c, rgb=rgb, alpha=alpha, background=_uniform(g, B, 3, H, W), d_image=_normal(g, B, 3, H, W))
        for k in ("rgb", "alpha", "background"):
            s[k].requires_grad_(True)
        return s
    R, V, S = c["R"], c["V"], c["S"]
    if c["dist"] == "normal":                                          # a head's logits
        logits = 2.0 * _normal(g, R, V)
    elif c["dist"] == "opacity":                                       # opacities of a trained scene: most inside [0, 1], some pushed out
        logits = _uniform(g, R, V) + 0.15 * _normal(g, R, V)
    else:                                                              # log of each layer's weight in a pixel; -inf where it is not there
        logits = _uniform(g, R, V).log_()
        gone = _uniform(g, R, V) < 0.3
        gone |= _uniform(g, R, 1) < 0.02
        logits.masked_fill_(gone, -math.inf)
    s = dict(case=c, logits=logits.to(DTYPES[c["dtype"]]), uniforms=_uniform(g, R, S, dtype=torch.float64 if c["dist"] == "opacity" else torch.float32))
    if c["rows"]:
        s.update(temperature=c["temperature"] * (0.5 + _uniform(g, R)), top_k=torch.randint(1, 2 * max(1, c["top_k"]) + 1, (R,), generator=g, device="cuda", dtype=torch.int32) * int(c["top_k"] > 0),
                 top_p=(c["top_p"] - 0.1 * _uniform(g, R) * float(c["top_p"] < 1.0)).to(torch.float32), min_p=c["min_p"] * _uniform(g, R))
    else:
        s.update(temperature=c["temperature"], top_k=c["top_k"], top_p=c["top_p"], min_p=c["min_p"])
    return s


# ------------------------------------------------------------------------------------------------------------ one pass
def run(s):
    op = s["case"]["op"]
    if own:
        return {"step": _own_step, "scan": _own_scan, "layers": _own_layers, "draw": _own_draw}[op](s)
    return {"step": _plain_step, "scan": _plain_scan, "layers": _plain_layers, "draw": _plain_draw}[op](s)


def _own_step(s):
    from gaussian_splatting_amd.recurrence import gated_step
    return gated_step(s["state"], s["gate"], s["x"], form=s["case"]["form"])


def _own_scan(s):
    from gaussian_splatting_amd.recurrence import gated_scan
    c = s["case"]
    states, last = gated_scan(s["gate"], s["x"], s["initial"], lengths=s["lengths"], form=c["form"], reverse=c["reverse"])
    if not c["train"]:
        return dict(states=states, last=last)
    d_gate, d_x, d_initial = torch.autograd.grad((states, last), (s["gate"], s["x"], s["initial"]), (s["d_states"], s["d_last"]))
    return dict(states=states, last=last, d_gate=d_gate, d_x=d_x, d_initial=d_initial)


def _own_layers(s):
    from gaussian_splatting_amd.render import composite_layers
    image = composite_layers(s["rgb"], s["alpha"], s["background"], straight=s["case"]["straight"])
    d_rgb, d_alpha, d_background = torch.autograd.grad(image, (s["rgb"], s["alpha"], s["background"]), s["d_image"])
    return dict(image=image, d_rgb=d_rgb, d_alpha=d_alpha, d_background=d_background)


def _own_draw(s):
    from gaussian_splatting_amd.sampling import sample
    indices, logprobs = sample(s["logits"], s["uniforms"], temperature=s["temperature"], top_k=s["top_k"], top_p=s["top_p"], min_p=s["min_p"], return_logprobs=True)
    return dict(indices=indices, logprobs=logprobs)


# ------------------------------------------------------------------------------------------------------------ plain forms
def _coefficients(form, gate, x):
    """h_t = a h_(t-1) + b"""
    if form == "linear":
        return gate, x
    return 1.0 - gate, (gate * x if form == "blend" else x)


def _doubling(a, b):
    """Inclusive scan of h_t = a_t h_(t-1) + b_t from h_(-1) = 0 along axis 1, by spans that double."""
    span, T = 1, a.shape[1]
    while span < T:
        b = torch.cat([b[:, :span], torch.addcmul(b[:, span:], a[:, span:], b[:, :-span])], 1)
        a = torch.cat([a[:, :span], a[:, span:] * a[:, :-span]], 1)
        span *= 2
    return b


def _states(a, b, initial):
    return _doubling(a, torch.cat([torch.addcmul(b[:, :1], a[:, :1], initial[:, None]), b[:, 1:]], 1))


def _adjoint(a, d):
    """g_t = d_t + a_(t+1) g_(t+1)"""
    after = torch.cat([a[:, 1:], torch.zeros_like(a[:, :1])], 1)
    return _doubling(after.flip(1), d.flip(1)).flip(1)


def _plain_step(s):
    with torch.no_grad():
        a, b = _coefficients(s["case"]["form"], s["gate"].float(), s["x"].float())
        return s["state"].mul_(a).add_(b)


def _plain_scan(s):
    with torch.no_grad():
        c = s["case"]
        t = DTYPES[c["dtype"]]
        gate, x = s["gate"].float(), s["x"].float()
        if c["reverse"]:
            gate, x = gate.flip(1), x.flip(1)
        a, b = _coefficients(c["form"], gate, x)
        inside = None
        if s["lengths"] is not None:                                   # a step behind the sequence's end changes nothing
            at = torch.arange(c["T"], device=gate.device)
            inside = ((at if not c["reverse"] else at.flip(0))[None, :] < s["lengths"][:, None])[..., None]
            a, b = torch.where(inside, a, 1.0), torch.where(inside, b, 0.0)
        h = _states(a, b, s["initial"])
        out = dict(states=h if inside is None else torch.where(inside, h, 0.0), last=h[:, -1])
        if c["train"]:
            d = s["d_states"].float()
            d = d.flip(1) if c["reverse"] else d
            d = d.clone() if inside is None else torch.where(inside, d, 0.0)
            d[:, -1] += s["d_last"]
            g = _adjoint(a, d)
            before = torch.cat([s["initial"][:, None], h[:, :-1]], 1)
            d_x = gate * g if c["form"] == "blend" else g
            d_gate = g * before if c["form"] == "linear" else g * (x - before) if c["form"] == "blend" else -g * before
            if inside is not None:
                d_x, d_gate = torch.where(inside, d_x, 0.0), torch.where(inside, d_gate, 0.0)
            out.update(d_gate=d_gate, d_x=d_x, d_initial=a[:, 0] * g[:, 0])
        for k in ("states", "d_gate", "d_x"):
            if k in out:
                out[k] = (out[k].flip(1) if c["reverse"] else out[k]).to(t)
        return out


def _plain_layers(s):
    with torch.no_grad():
        # layers in front have the lower number: the recurrence goes from the last layer to the first
        rgb, alpha = s["rgb"].flip(0).transpose(0, 1), s["alpha"].flip(0).transpose(0, 1)
        a, b = _coefficients("blend" if s["case"]["straight"] else "over", alpha, rgb)
        a = a.expand_as(b)
        h = _states(a, b, s["background"])
        d = torch.zeros_like(h)
        d[:, -1] = s["d_image"]
        g = _adjoint(a, d)
        before = torch.cat([s["background"][:, None], h[:, :-1]], 1)
        d_rgb = alpha * g if s["case"]["straight"] else g
        d_alpha = (g * ((rgb - before) if s["case"]["straight"] else -before)).sum(2, keepdim=True)
        return dict(image=h[:, -1].contiguous(), d_rgb=d_rgb.transpose(0, 1).flip(0), d_alpha=d_alpha.transpose(0, 1).flip(0), d_background=a[:, 0] * g[:, 0])


def _column(v, like):
    """A setting of one row or of all, in the 32 bits that it has as an argument, as a column of 64-bit numbers."""
    if torch.is_tensor(v):
        return v.to(torch.float32).double()[:, None]
    return torch.full((like.shape[0], 1), v, dtype=torch.float32, device=like.device).double()


def _plain_draw(s):
    logits = s["logits"].double()
    R, V = logits.shape
    logits = torch.where(torch.isnan(logits), -math.inf, logits)
    top = logits.amax(1, keepdim=True)
    T, p, min_p = (_column(s[k], logits) for k in ("temperature", "top_p", "min_p"))
    k = s["top_k"].long()[:, None] if torch.is_tensor(s["top_k"]) else torch.full((R, 1), s["top_k"], dtype=torch.long, device=logits.device)
    w = torch.where(logits == top, 1.0, torch.exp((logits - top) / T))     # weights as shares of the largest
    w = torch.where(torch.isneginf(logits), 0.0, w)
    order = torch.sort(logits, dim=1, descending=True, stable=True).indices
    ranked = w.gather(1, order)
    place = torch.arange(V, device=logits.device)[None, :]
    keep = (place < k) | (k <= 0)
    ranked_kept = torch.where(keep, ranked, 0.0)
    before = torch.cumsum(ranked_kept, 1) - ranked_kept
    keep &= (before < p * ranked_kept.sum(1, keepdim=True)) | (p >= 1.0)
    keep &= ranked >= min_p
    w = torch.where(torch.zeros_like(keep).scatter_(1, order, keep), w, 0.0)
    mass = torch.cumsum(w, 1)
    total = mass[:, -1:].contiguous()
    indices = torch.searchsorted(mass, s["uniforms"].double() * total, right=True)
    indices = torch.minimum(indices, torch.full_like(indices, V - 1))
    logprobs = torch.log(w.gather(1, indices) / total).to(torch.float32)
    nothing = total == 0.0
    return dict(indices=torch.where(nothing, -1, indices), logprobs=torch.where(nothing, -math.inf, logprobs))


# ------------------------------------------------------------------------------------------------------------ the least work
def work(case):
    c = case
    if c["op"] == "step":
        n, e = c["B"] * c["D"], DTYPES[c["dtype"]].itemsize
        return {"bytes": n * (2 * e + 8), "flops": 3 * n}
    if c["op"] == "scan":
        n, e = c["B"] * c["T"] * c["D"], DTYPES[c["dtype"]].itemsize
        share = 0.5 if c["ragged"] else 1.0                            # steps behind the end of a sequence are not read
        moved = (2 * share + 1) * n * e
        if c["train"]:                                                 # and the states' gradient read, two gradients written
            moved += (share + 2) * n * e
        return {"bytes": moved + 8 * c["B"] * c["D"] * (2 if c["train"] else 1), "flops": (8 if c["train"] else 3) * n * share}
    if c["op"] == "layers":
        n = c["B"] * c["H"] * c["W"]
        return {"bytes": 4 * n * (8 * c["L"] + 12), "flops": n * c["L"] * 3 * 8}
    n = c["R"] * c["V"]
    return {"bytes": n * DTYPES[c["dtype"]].itemsize + c["R"] * c["S"] * ((8 if c["dist"] == "opacity" else 4) + 12), "flops": 30 * n}


# ------------------------------------------------------------------------------------------------------------ the definition
def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        if case["op"] == "draw":
            return _exact_draw(s)
        return {"step": _exact_step, "scan": _exact_scan, "layers": _exact_layers}[case["op"]](s)


def _exact_step(s):
    h, z, x = s["state"].double(), s["gate"].double(), s["x"].double()
    form = s["case"]["form"]
    return z * h + x if form == "linear" else (1 - z) * h + (z * x if form == "blend" else x)


def _walk(form, gate, x, h, alive, d_states, d_last):
    """One step after the other in 64 bits: lists over the steps of gate (B, ...), x, whether the step belongs to the sequence, the gradient of each state."""
    states, before = [], []
    for z, v, ok in zip(gate, x, alive):
        before.append(h)
        n = z * h + v if form == "linear" else (1 - z) * h + (z * v if form == "blend" else v)
        h = n if ok is None else torch.where(ok, n, h)
        states.append(h if ok is None else torch.where(ok, h, 0.0))
    if d_last is None:
        return states, h
    g, d_gate, d_x = d_last, [None] * len(states), [None] * len(states)
    for t in range(len(states) - 1, -1, -1):
        z, v, ok = gate[t], x[t], alive[t]
        here = g if d_states is None else g + (d_states[t] if ok is None else torch.where(ok, d_states[t], 0.0))
        dz = here * before[t] if form == "linear" else here * (v - before[t]) if form == "blend" else -here * before[t]
        dv = z * here if form == "blend" else here
        back = (z if form == "linear" else 1 - z) * here
        g = back if ok is None else torch.where(ok, back, g)
        d_gate[t], d_x[t] = (dz, dv) if ok is None else (torch.where(ok, dz, 0.0), torch.where(ok, dv, 0.0))
    return states, h, d_gate, d_x, g


def _exact_scan(s):
    c = s["case"]
    steps = list(range(c["T"]))
    steps = steps[::-1] if c["reverse"] else steps
    gate, x = s["gate"].double(), s["x"].double()
    alive = [None if s["lengths"] is None else (s["lengths"] > t)[:, None] for t in steps]
    d_states = s["d_states"].double() if c["train"] else None
    got = _walk(c["form"], [gate[:, t] for t in steps], [x[:, t] for t in steps], s["initial"].double(), alive,
                [d_states[:, t] for t in steps] if c["train"] else None, s["d_last"].double() if c["train"] else None)
    whole = lambda v: torch.stack(v[::-1] if c["reverse"] else v, 1)  # noqa: E731
    out = dict(states=whole(got[0]), last=got[1])
    if c["train"]:
        out.update(d_gate=whole(got[2]), d_x=whole(got[3]), d_initial=got[4])
    return out


def _exact_layers(s):
    rgb, alpha = s["rgb"].double(), s["alpha"].double()
    L = rgb.shape[0]
    got = _walk("blend" if s["case"]["straight"] else "over", [alpha[t] for t in range(L - 1, -1, -1)], [rgb[t] for t in range(L - 1, -1, -1)],
                s["background"].double(), [None] * L, None, s["d_image"].double())
    return dict(image=got[1], d_rgb=torch.stack(got[3][::-1]), d_alpha=torch.stack(got[2][::-1]).sum(2, keepdim=True), d_background=got[4])


def _exact_draw(s):
    """Row by row (blocks of rows where they are short): ranks from a sort of (logit, place), whole prefixes of the ranking kept, and the draw by counting."""
    logits = s["logits"].double().cpu().numpy()
    u = s["uniforms"].double().cpu().numpy()
    R, V = logits.shape
    each = lambda v, t: np.broadcast_to(v.cpu().numpy() if torch.is_tensor(v) else np.asarray(v), (R,)).astype(t)  # noqa: E731
    T, p, min_p = (each(s[k], np.float32).astype(np.float64) for k in ("temperature", "top_p", "min_p"))
    top_k = each(s["top_k"], np.int64)
    indices, logprobs = np.empty(u.shape, np.int64), np.empty(u.shape, np.float64)
    rows = max(1, min(R, (1 << 22) // V))
    for r in range(0, R, rows):
        l, q = logits[r:r + rows], slice(r, r + rows)
        best = np.max(l, 1, keepdims=True)
        with np.errstate(invalid="ignore", divide="ignore"):
            w = np.exp((l - best) / T[q, None])
        w[np.isneginf(l)] = 0.0
        order = np.argsort(-l, 1, kind="stable")
        ranked = np.take_along_axis(w, order, 1)
        count = np.where(top_k[q] > 0, np.minimum(top_k[q], V), V)[:, None]
        at = np.arange(V)[None]
        ranked[np.broadcast_to(at, ranked.shape) >= count] = 0.0
        run_up = np.cumsum(ranked, 1)
        wanted = p[q, None] * run_up[:, -1:]
        reach = 1 + np.sum(run_up < wanted, 1, keepdims=True)          # the fewest places whose mass reaches the share
        count = np.where(p[q, None] < 1.0, np.minimum(count, reach), count)
        count = np.minimum(count, np.sum(ranked >= min_p[q, None], 1, keepdims=True))
        kept = np.zeros(w.shape, bool)
        np.put_along_axis(kept, order, np.broadcast_to(at, w.shape) < count, 1)
        w = np.where(kept, w, 0.0)
        c = np.cumsum(w, 1)
        for i in range(len(l)) if V > 512 else ():
            indices[r + i] = np.searchsorted(c[i], u[r + i] * c[i, -1], side="right")
        if V <= 512:
            indices[q] = np.stack([np.sum(c <= u[q, j:j + 1] * c[:, -1:], 1) for j in range(u.shape[1])], 1)
        at = np.minimum(indices[q], V - 1)
        with np.errstate(divide="ignore", invalid="ignore"):
            logprobs[q] = np.log(np.take_along_axis(w, at, 1)) - np.log(c[:, -1:])
        indices[q] = np.where(c[:, -1:] > 0.0, at, -1)
        logprobs[q] = np.where(c[:, -1:] > 0.0, logprobs[q], -np.inf)
    return dict(indices=torch.from_numpy(indices), logprobs=torch.from_numpy(logprobs))
