"""The gated scan (gaussian_splatting_amd.recurrence, csrc/gsx_gated.hip) against the recurrence in 64 bits, step by step, with a bound
that the same walk computes: every operation of the kernel rounds by at most half a step of 32 bits (U = 2^-24 relative), every output
by half a step of its own type."""
import pytest
import torch

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def _half_step(t, v):
    """how far rounding v to t may move it: half a step, or half of the smallest number"""
    fi = torch.finfo(t)
    return v.abs() * (fi.eps / 2) + fi.smallest_normal * (fi.eps / 2)


def walk(form, gate, x, initial, lengths, reverse, d_states=None, d_last=None):
    """64-bit values and bounds of the error of a 32-bit walk.  gate (B, T, D), x (B, T, P, D), all double.
    h = fma(a, h, m x): a = 1 - z rounds once, m x once, the fma once: e' = |a| e + U(2 |a h| + 2 |m x|) and second-order terms, 4 U in all.
    g = d + c rounds once; c' = a g: two roundings; dx = m g: one more; dz: the product with h or x - h, summed over the planes."""
    B, T, P, D = x.shape
    order = list(range(T))[::-1] if reverse else list(range(T))
    h, e = initial.clone(), torch.zeros_like(initial)
    states, e_states = torch.zeros_like(x), torch.zeros_like(x)
    before = {}
    for t in order:
        z = gate[:, t, None]
        a, m = (z, torch.ones_like(z)) if form == "linear" else (1 - z, z if form == "blend" else torch.ones_like(z))
        ok = torch.ones(B, dtype=torch.bool, device=x.device) if lengths is None else lengths > t
        before[t] = (h, e, a, m, ok[:, None, None])
        b = torch.where(ok[:, None, None], m * x[:, t], 0.0)
        hn = torch.where(ok[:, None, None], a * h + b, h)
        en = torch.where(ok[:, None, None], a.abs() * e + 4 * U * ((a * h).abs() + b.abs()), e)
        h, e = hn, en
        states[:, t], e_states[:, t] = torch.where(ok[:, None, None], h, 0.0), torch.where(ok[:, None, None], e, 0.0)
    out = dict(states=(states, e_states), last=(h, e))
    if d_last is None and d_states is None:
        return out
    c = torch.zeros_like(h) if d_last is None else d_last.clone()
    ec = torch.zeros_like(c)
    dg, eg_, dx, ex = torch.zeros_like(gate), torch.zeros_like(gate), torch.zeros_like(x), torch.zeros_like(x)
    for t in order[::-1]:
        hb, eb, a, m, ok = before[t]
        g = c if d_states is None else c + d_states[:, t]
        eg = ec + 2 * U * g.abs()
        v = hb if form == "linear" else (x[:, t] - hb if form == "blend" else -hb)
        ev = eb + (2 * U * v.abs() if form == "blend" else 0.0)
        dg[:, t] = torch.where(ok, g * v, 0.0).sum(1)
        eg_[:, t] = torch.where(ok, g.abs() * ev + eg * v.abs() + eg * ev + 8 * U * (g * v).abs(), 0.0).sum(1)
        dx[:, t] = torch.where(ok, m * g, 0.0)
        ex[:, t] = torch.where(ok, m.abs() * eg + 2 * U * (m * g).abs(), 0.0)
        ec = torch.where(ok, a.abs() * eg + 4 * U * (a * g).abs(), ec)
        c = torch.where(ok, a * g, c)
    out.update(d_gate=(dg, eg_), d_x=(dx, ex), d_initial=(c, ec))
    return out


def close(got, want, t, what):
    v, e = want
    assert got.dtype == t and got.shape == v.shape, (what, got.dtype, got.shape)
    off = (got.double() - v).abs()
    allowed = e * 1.01 + _half_step(t, v.abs() + e) + 1e-38
    assert bool((off <= allowed).all()), (what, float((off / allowed).max()))


def make(B, T, P, D, t, form, seed, ragged=False, with_initial=True):
    g = torch.Generator(device="cuda").manual_seed(seed)
    rn = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    keep = torch.sigmoid(1.5 + 2 * rn(B, T, D))
    gate = (keep if form == "linear" else 1 - keep).to(t)
    x = (rn(B, T, P, D) if P > 1 else rn(B, T, D)).to(t)
    initial = (rn(B, P, D) if P > 1 else rn(B, D)) if with_initial else None
    lengths = torch.randint(0, T + 1, (B,), generator=g, device="cuda", dtype=torch.int32) if ragged else None
    return gate, x, initial, lengths, rn(*x.shape).to(t), rn(*(x.shape[:1] + x.shape[2:]))


def check(gate, x, initial, lengths, d_states, d_last, t, form, reverse, return_states=True):
    from gaussian_splatting_amd import gated_scan
    four = lambda v: v if v is None or x.dim() == 4 else v.unsqueeze(-2)  # noqa: E731
    i64 = torch.zeros(x.shape[:1] + x.shape[2:], dtype=torch.float64, device=x.device) if initial is None else initial.double()
    want = walk(form, gate.double(), four(x.double()), four(i64), lengths, reverse, four(d_states.double()) if return_states else None, four(d_last.double()))
    leaves = [v.detach().requires_grad_(True) for v in (gate, x) + (() if initial is None else (initial,))]
    states, last = gated_scan(leaves[0], leaves[1], leaves[2] if initial is not None else None, lengths=lengths, form=form, reverse=reverse, return_states=return_states)
    pick = lambda k: tuple(v if x.dim() == 4 or k == "d_gate" else v.squeeze(-2) for v in want[k])  # noqa: E731
    close(last, pick("last"), torch.float32, "last")
    if return_states:
        close(states, pick("states"), t, "states")
        got = torch.autograd.grad((states, last), leaves, (d_states, d_last))
    else:
        assert states is None
        got = torch.autograd.grad(last, leaves, d_last)
    close(got[0], pick("d_gate"), t, "d_gate")
    close(got[1], pick("d_x"), t, "d_x")
    if initial is not None:
        close(got[2], pick("d_initial"), torch.float32, "d_initial")


SHAPES = [(1, 1, 1, 1), (1, 1, 1, 64), (2, 15, 1, 3), (1, 16, 1, 130), (3, 17, 1, 65), (2, 33, 2, 7), (1, 8, 3, 129), (2, 9, 4, 33), (5, 100, 1, 2), (1, 700, 1, 20),
          (2, 1500, 3, 5), (1, 4099, 1, 66), (3, 2049, 1, 34)]


@pytest.mark.parametrize("shape", SHAPES, ids=str)
@pytest.mark.parametrize("form,dtype,reverse,ragged", [("linear", "f32", False, False), ("blend", "bf16", False, True), ("over", "f16", True, True), ("over", "f32", True, False),
                                                       ("blend", "f32", True, True), ("linear", "bf16", True, False)])
def test_scan_and_gradients_against_64_bits(shape, form, dtype, reverse, ragged):
    B, T, P, D = shape
    a = make(B, T, P, D, DT[dtype], form, 17 + T, ragged, with_initial=(T % 2 == 0) or ragged)
    check(*a, DT[dtype], form, reverse, return_states=not (P == 3))


@pytest.mark.parametrize("shape", [(1, 3, 1, 300001), (40, 5, 1, 4096), (64, 130, 1, 1024)], ids=str)
def test_wide_scans(shape):
    B, T, P, D = shape
    a = make(B, T, P, D, torch.bfloat16, "linear", 3, ragged=B > 1)
    check(*a, torch.bfloat16, "linear", False)


def test_long_scan_splits_the_steps():
    a = make(1, 20011, 1, 3, torch.float32, "linear", 5)
    check(*a, torch.float32, "linear", False)


def test_strides_offsets_and_odd_alignment():
    """views of larger arrays: steps first, a plane in between, one element off every boundary, expanded gates and gradients"""
    from gaussian_splatting_amd import gated_scan
    g = torch.Generator(device="cuda").manual_seed(2)
    for t in (torch.float32, torch.bfloat16):
        B, T, D = 3, 37, 50
        big_g = torch.rand(T, B, 2, D + 3, generator=g, device="cuda").to(t)
        big_x = torch.randn(T, B, 2, D + 3, generator=g, device="cuda").to(t)
        for off in (0, 1, 2):
            gate, x = big_g[:, :, 1, off:off + D].transpose(0, 1), big_x[:, :, 0, off:off + D].transpose(0, 1)
            d = torch.randn(B, T, 1, generator=g, device="cuda").to(t).expand(B, T, D)
            check(gate, x, None, None, d, torch.zeros(B, D, device="cuda"), t, "linear", False)
        gate, x = big_g[:, :1, 1, :D].transpose(0, 1).expand(B, T, D), big_x[:, :, 0, :D].transpose(0, 1)
        want = walk("over", gate.double(), x.double()[:, :, None], torch.zeros(B, 1, D, dtype=torch.float64, device="cuda"), None, False)
        states, last = gated_scan(gate, x, form="over")
        close(states, tuple(v[:, :, 0] for v in want["states"]), t, "states")
        # channels that are not consecutive are laid out first
        xt = x.transpose(1, 2).contiguous().transpose(1, 2)
        assert torch.equal(gated_scan(gate, xt, form="over")[0], states)


def test_what_lies_behind_a_sequence_is_not_read():
    from gaussian_splatting_amd import gated_scan
    for reverse in (False, True):
        gate, x, initial, _, d, dl = make(4, 40, 1, 9, torch.float32, "blend", 8)
        lengths = torch.tensor([0, 7, 40, 99], dtype=torch.int32, device="cuda")
        outs = []
        for poison in (0.0, float("nan"), float("inf")):
            gz, xz, dz = gate.clone(), x.clone(), d.clone()
            for b, n in enumerate((0, 7, 40, 40)):
                gz[b, n:], xz[b, n:], dz[b, n:] = poison, poison, poison
            leaves = [v.requires_grad_(True) for v in (gz, xz, initial.clone())]
            s, l = gated_scan(*leaves, lengths=lengths, form="blend", reverse=reverse)
            outs.append((s, l) + torch.autograd.grad((s, l), leaves, (dz, dl)))
        for o in outs[1:]:
            for a, b in zip(outs[0], o):
                assert torch.equal(a, b)
        s, l, dg, dx, di = outs[0]
        assert torch.equal(l[0], initial[0]) and torch.equal(di[0], dl[0]) and not s[0].any() and not s[1, 7:].any() and not dg[1, 7:].any() and not dx[0].any()


def test_no_steps_and_empty_batches():
    from gaussian_splatting_amd import gated_scan
    i = torch.randn(2, 5, device="cuda", requires_grad=True)
    z = torch.zeros(2, 0, 5, device="cuda", requires_grad=True)
    s, l = gated_scan(z, z.detach(), i)
    assert s.shape == (2, 0, 5) and torch.equal(l, i)
    (di,) = torch.autograd.grad(l.sum(), i)
    assert torch.equal(di, torch.ones_like(i))
    for shape in ((0, 4, 5), (2, 4, 0)):
        z = torch.zeros(shape, device="cuda")
        s, l = gated_scan(z, z)
        assert s.shape == shape and l.shape == (shape[0], shape[2])


def test_resets_and_growing_gates():
    """a zero gate forgets exactly; gates above one grow as far as 32 bits go, also where whole spans of steps multiply to more"""
    from gaussian_splatting_amd import gated_scan
    gate, x, initial, _, _, _ = make(1, 3001, 1, 40, torch.float32, "linear", 4)
    gate[:, 1000] = 0.0
    states, _ = gated_scan(gate, x, initial)
    again, _ = gated_scan(gate[:, 1000:], x[:, 1000:])
    want = walk("linear", gate[:, 1000:].double(), x[:, 1000:].double()[:, :, None], torch.zeros(1, 1, 40, dtype=torch.float64, device="cuda"), None, False)
    close(states[:, 1000:], tuple(v[:, :, 0] for v in want["states"]), torch.float32, "states")
    close(again, tuple(v[:, :, 0] for v in want["states"]), torch.float32, "again")
    gate = torch.full((1, 6000, 8), 1.25, device="cuda")
    x = torch.zeros(1, 6000, 8, device="cuda")
    x[:, 5900] = 1.0                                       # nothing before it: 1.25^n leaves 32 bits, and times a zero state is a zero
    states, last = gated_scan(gate, x)
    assert not states[:, :5900].any() and torch.isfinite(states).all()
    want = torch.tensor(1.25, dtype=torch.float64) ** 99
    assert bool(((last.double() - want.cuda()).abs() <= 100 * 4 * U * want.cuda()).all())


def test_a_call_in_pieces_equals_one_call():
    from gaussian_splatting_amd import gated_scan, gated_step
    gate, x, initial, _, _, _ = make(2, 61, 1, 48, torch.float32, "blend", 11)
    states, last = gated_scan(gate, x, initial, form="blend")
    h, parts = initial, []
    for a, b in ((0, 1), (1, 20), (20, 61)):
        s, h = gated_scan(gate[:, a:b], x[:, a:b], h, form="blend")
        parts.append(s)
    assert torch.equal(torch.cat(parts, 1), states) and torch.equal(h, last)
    h = initial.clone()
    for t in range(61):
        assert gated_step(h, gate[:, t].contiguous(), x[:, t].contiguous(), form="blend") is h
        assert torch.equal(h, states[:, t])


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("form", ["linear", "blend", "over"])
@pytest.mark.parametrize("shape", [(1,), (3, 5), (64, 2048), (7, 33, 4)], ids=str)
def test_step(dtype, form, shape):
    from gaussian_splatting_amd import gated_step
    t = DT[dtype]
    g = torch.Generator(device="cuda").manual_seed(1)
    state, x = torch.randn(shape, generator=g, device="cuda"), torch.randn(shape, generator=g, device="cuda").to(t)
    z = torch.rand(shape, generator=g, device="cuda").to(t)
    a, m = (z.double(), 1.0) if form == "linear" else (1 - z.double(), z.double() if form == "blend" else 1.0)
    want, size = a * state.double() + m * x.double(), (a * state.double()).abs() + (m * x.double()).abs()
    version = state._version
    gated_step(state, z, x, form=form)
    assert state._version > version
    assert bool(((state.double() - want).abs() <= 4 * U * size + 1e-38).all())
    # one element off the boundary that wide loads want
    buf = torch.zeros(state.numel() + 1, device="cuda")
    odd = buf[1:].view(shape).copy_(torch.ones(shape, device="cuda"))
    even = torch.ones(shape, device="cuda")
    assert torch.equal(gated_step(odd, z, x, form=form), gated_step(even, z, x, form=form)) and float(buf[0]) == 0.0


def test_gradients_against_differences():
    """central differences of the 64-bit walk, 1e-6 wide: off by 1e-12 of the third derivative and 1e-10 of rounding, against 32 bits"""
    from gaussian_splatting_amd import gated_scan
    for form in ("linear", "blend", "over"):
        gate, x, initial, lengths, d, dl = make(2, 21, 3, 5, torch.float32, form, 23, ragged=True)
        leaves = [v.requires_grad_(True) for v in (gate, x, initial)]
        s, l = gated_scan(*leaves, lengths=lengths, form=form)
        grads = torch.autograd.grad((s, l), leaves, (d, dl))
        loss = lambda *v: float((lambda o: (o["states"][0] * d.double()).sum() + (o["last"][0] * dl.double()).sum())(walk(form, *v, lengths, False)))  # noqa: E731
        gen = torch.Generator(device="cuda").manual_seed(0)
        base = [v.detach().double() for v in leaves]
        for k in range(3):
            v = torch.randn(base[k].shape, generator=gen, device="cuda", dtype=torch.float64)
            shift = lambda e: [b + e * v if j == k else b for j, b in enumerate(base)]  # noqa: E731
            diff = (loss(*shift(1e-6)) - loss(*shift(-1e-6))) / 2e-6
            dot, size = float((grads[k].double() * v).sum()), float((grads[k].double() * v).abs().sum())
            assert abs(dot - diff) <= 1e-5 * size, (form, k, dot, diff)


def test_the_same_bits_on_another_stream_and_every_time():
    from gaussian_splatting_amd import gated_scan
    gate, x, initial, lengths, d, dl = make(2, 3000, 1, 70, torch.bfloat16, "linear", 6, ragged=True)
    def once():
        leaves = [v.detach().requires_grad_(True) for v in (gate, x, initial)]
        s, l = gated_scan(*leaves, lengths=lengths)
        return (s, l) + torch.autograd.grad((s, l), leaves, (d, dl))
    first = once()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = once()
    torch.cuda.current_stream().wait_stream(side)
    for a, b in zip(first, other):
        assert torch.equal(a, b)


def test_captured_and_replayed():
    from gaussian_splatting_amd import gated_scan, gated_step
    gate, x, initial, _, d, dl = make(2, 1200, 1, 66, torch.float32, "linear", 6)
    state = torch.zeros_like(initial)
    leaves = [v.requires_grad_(True) for v in (gate, x, initial)]
    def work():
        s, l = gated_scan(*leaves)
        return (s, l) + torch.autograd.grad((s, l), leaves, (d, dl)) + (gated_step(state, gate[:, 0].detach(), x[:, 0].detach()),)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        work()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    state.zero_()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = work()
    for n in range(4):
        with torch.no_grad():
            x.copy_(torch.randn(x.shape, device="cuda"))
            gate.copy_(torch.rand(gate.shape, device="cuda"))
        state.fill_(float(n))
        graph.replay()
        torch.cuda.synchronize()
        got = [v.clone() for v in out]
        state.fill_(float(n))
        for a, b in zip(got, work()):
            assert torch.equal(a, b), n


def test_layers_of_real_renders_and_their_gradients():
    """two scenes rendered apart and laid over each other, down to the Gaussians' gradients, against the formula on the same renders"""
    from gaussian_splatting_amd import GaussianSplat, composite_layers
    from gaussian_splatting_amd.scenes import pose_tz
    torch.manual_seed(0)
    scenes = [GaussianSplat(400).cuda() for _ in range(3)]
    pose = torch.from_numpy(pose_tz(2.0))[None].cuda().expand(2, 4, 4)
    bg = torch.rand(2, 3, 40, 56, device="cuda")
    def grads(layer_over):
        outs = [m(pose, (40, 56)) for m in scenes]
        rgb, alpha = torch.stack([o["rendered_images"] for o in outs]), torch.stack([o["alpha"] for o in outs])
        image = layer_over(rgb, alpha)
        w = torch.linspace(-1, 1, image.numel(), device="cuda").view_as(image)
        return [image] + list(torch.autograd.grad((image * w).sum(), [m.features for m in scenes] + [m.positions for m in scenes], allow_unused=True))
    def plain(rgb, alpha):
        c = bg.double()
        for k in (2, 1, 0):
            c = (1 - alpha[k].double()) * c + rgb[k].double()
        return c.float()
    ours = grads(lambda rgb, alpha: composite_layers(rgb, alpha, bg))
    want = grads(plain)
    assert float((ours[0] - want[0]).abs().max()) <= 16 * U * float(want[0].abs().max() + 1)
    for a, b in zip(ours[1:], want[1:]):
        # the gradients of the image reach the splats through the render's own backward: linear in what differs by a few roundings
        assert float((a - b).abs().max()) <= 1e-4 * float(b.abs().max()) + 1e-9


@pytest.mark.parametrize("straight", [False, True])
@pytest.mark.parametrize("P", [1, 3, 4])
def test_layers_against_64_bits(straight, P):
    from gaussian_splatting_amd import composite_layers
    g = torch.Generator(device="cuda").manual_seed(9)
    n, B, H, W = 11, 2, 13, 17
    alpha = torch.rand(n, B, 1, H, W, generator=g, device="cuda", requires_grad=True)
    rgb = torch.rand(n, B, P, H, W, generator=g, device="cuda", requires_grad=True)
    bg = torch.rand(B, P, H, W, generator=g, device="cuda", requires_grad=True)
    d = torch.randn(B, P, H, W, generator=g, device="cuda")
    want = walk("blend" if straight else "over", alpha.detach().double().reshape(n, B, H * W).transpose(0, 1), rgb.detach().double().reshape(n, B, P, H * W).transpose(0, 1),
                bg.detach().double().reshape(B, P, -1), None, True, None, d.double().reshape(B, P, -1))
    image = composite_layers(rgb, alpha, bg, straight=straight)
    got = torch.autograd.grad(image, (alpha, rgb, bg), d)
    close(image.reshape(B, P, -1), want["last"], torch.float32, "image")
    close(got[0].reshape(n, B, -1).transpose(0, 1), want["d_gate"], torch.float32, "d_alpha")
    close(got[1].reshape(n, B, P, -1).transpose(0, 1), want["d_x"], torch.float32, "d_rgb")
    close(got[2].reshape(B, P, -1), want["d_initial"], torch.float32, "d_background")
    assert torch.equal(composite_layers(rgb, alpha, straight=straight), composite_layers(rgb, alpha, torch.zeros_like(bg), straight=straight))


def test_a_trace_over_views_picks_the_points():
    """the two operators as they are used together: the visible share of every Gaussian in each view of an orbit, a decayed trace of it, and dense
    points drawn from the trace"""
    from gaussian_splatting_amd import GaussianSplat, gated_scan
    from gaussian_splatting_amd.scenes import create_orbit_poses
    torch.manual_seed(1)
    n, V = 3000, 9
    m = GaussianSplat(n).cuda()
    poses = torch.from_numpy(create_orbit_poses(2.0, V, 30.0)).float().cuda()
    scores = torch.empty(1, V, n, device="cuda")
    for v in range(V):
        out = m(poses[v:v + 1], (48, 64))
        scores[0, v] = torch.autograd.grad(out["rendered_images"].sum(), m.features)[0].sum(1).abs()
    decay = torch.full((1, V, n), 0.8, device="cuda")
    _, trace = gated_scan(decay, scores, return_states=False)
    want = walk("linear", decay.double(), scores.double()[:, :, None], torch.zeros(1, 1, n, dtype=torch.float64, device="cuda"), None, False)["last"]
    close(trace, tuple(x[:, 0] for x in want), torch.float32, "trace")
    u = torch.rand(5000, device="cuda", dtype=torch.float64)
    pts = m.get_dense_points(5000, logits=torch.log(trace[0]), top_k=200, min_p=0.01, uniforms=u)
    rank = torch.sort(torch.log(trace[0]), descending=True, stable=True).indices[:200]
    w = torch.exp(torch.log(trace[0])[rank].double() - torch.log(trace[0]).max().double())
    kept, _ = torch.sort(rank[w >= torch.tensor(0.01).double().item()])
    lw = torch.exp(torch.log(trace[0])[kept].double() - torch.log(trace[0]).max().double())
    c = torch.cumsum(lw, 0)
    idx = kept[torch.searchsorted(c, u * c[-1], right=True)]
    assert torch.equal(pts, torch.cat([m.positions[idx], m.features[idx]], 1))


def test_offsets_beyond_32_bits():
    """more than 2^31 elements: the last channels to the last steps, forward and backward; the others are zero"""
    from gaussian_splatting_amd import gated_scan
    T, D, n = 2100, 1050000, 64
    gate, x = (torch.zeros(1, T, D, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    few_gate, few_x, _, _, d, dl = make(1, T, 1, n, torch.bfloat16, "linear", 40)
    gate[..., -n:], x[..., -n:] = few_gate, few_x
    want = walk("linear", few_gate.double(), few_x.double()[:, :, None], torch.zeros(1, 1, n, dtype=torch.float64, device="cuda"), None, False, d.double()[:, :, None], dl.double()[:, None])
    want = {k: v if k == "d_gate" else tuple(e.squeeze(-2) for e in v) for k, v in want.items()}
    states, last = gated_scan(gate.requires_grad_(True), x.requires_grad_(True))
    close(last[:, -n:], want["last"], torch.float32, "last")
    close(states[..., -n:], want["states"], torch.bfloat16, "states")
    assert not bool(last[:, :-n].any()) and not bool(states[:, -1, :-n].any())
    ds, dls = torch.zeros_like(states), torch.zeros_like(last)
    ds[..., -n:], dls[:, -n:] = d, dl
    got = torch.autograd.grad((states, last), (gate, x), (ds, dls))
    close(got[0][..., -n:], want["d_gate"], torch.bfloat16, "d_gate")
    close(got[1][..., -n:], want["d_x"], torch.bfloat16, "d_x")


def test_two_streams_at_once():
    from gaussian_splatting_amd import gated_scan
    sets = [make(2, 3000, 1, 70, torch.bfloat16, "linear", 6), make(1, 40, 3, 5000, torch.float32, "blend", 7)]
    def once(s, form):
        leaves = [v.detach().requires_grad_(True) for v in s[:3]]
        st, l = gated_scan(*leaves, form=form)
        return (st, l) + torch.autograd.grad((st, l), leaves, (s[4], s[5]))
    forms = ("linear", "blend")
    alone = [once(s, f) for s, f in zip(sets, forms)]
    streams = [torch.cuda.Stream() for _ in sets]
    torch.cuda.synchronize()
    outs = [[] for _ in sets]
    for _ in range(5):
        for st, s, f, o in zip(streams, sets, forms, outs):
            with torch.cuda.stream(st):
                o.append(once(s, f))
    torch.cuda.synchronize()
    for a, out in zip(alone, outs):
        for o in out:
            assert all(torch.equal(p, q) for p, q in zip(a, o))


def test_step_beside_and_upon_its_own_state():
    """gate and input next to the state in one buffer, and the state as its own gate or input; an overlap is refused"""
    from gaussian_splatting_amd import gated_step
    for n in (64, 67, 4096):
        buf = torch.rand(3 * n, device="cuda", generator=torch.Generator(device="cuda").manual_seed(n))
        s, g, x = buf[n:2 * n], buf[:n], buf[2 * n:]
        was = buf.double().clone()
        for gate, inp in ((g, x), (s, x), (g, s), (s, s)):
            buf.copy_(was.float())
            z, v, h = gate.double(), inp.double(), s.double()
            gated_step(s, gate, inp)
            assert bool(((s.double() - (z * h + v)).abs() <= 4 * U * ((z * h).abs() + v.abs())).all())
            assert torch.equal(buf[:n].double(), was[:n]) and torch.equal(buf[2 * n:].double(), was[2 * n:])
        for gate, inp in ((buf[n - 1:2 * n - 1], x), (g, buf[n + 1:2 * n + 1])):
            with pytest.raises(RuntimeError, match="gsx_gated_step"):
                gated_step(s, gate, inp)


def test_more_lanes_than_one_axis_of_a_launch():
    """more than 2^32 threads: every channel of every sequence, both ways, and one step.  One step of time, so the values are exact"""
    from gaussian_splatting_amd import gated_scan, gated_step
    B, D = 65537, 65536
    x = torch.randn(1, 1, D, device="cuda", generator=torch.Generator(device="cuda").manual_seed(1)).requires_grad_(True)
    gate = torch.full((1, 1, D), 0.5, device="cuda").expand(B, 1, D)
    _, last = gated_scan(gate, x.expand(B, 1, D), return_states=False)
    for b in range(0, B, 4096):
        assert bool((last[b:b + 4096] == x[0]).all()), b
    (dx,) = torch.autograd.grad(last, x, torch.ones(1, D, device="cuda").expand(B, D))
    assert bool((dx == float(B)).all())                              # a sum of B ones
    del last, dx
    n = (1 << 32) + 257                                              # odd: a lane per element
    half = torch.full((n,), 0.5, dtype=torch.bfloat16, device="cuda")
    state = torch.full((n,), 2.0, device="cuda")
    state[-1] = 4.0
    gated_step(state, half, half)
    assert float(state[-1]) == 2.5
    state[-1] = 1.5
    for i in range(0, n, 1 << 28):
        assert bool((state[i:i + (1 << 28)] == 1.5).all()), i


@pytest.mark.parametrize("form", ["linear", "blend", "over"])
def test_infinities_stay_where_the_walk_has_them(form):
    """an infinite state outlives gates whose product leaves 64 bits, also across spans that are walked apart; a zero gate makes it a NaN"""
    from gaussian_splatting_amd import gated_scan
    inf, T, D = float("inf"), 9001, 8
    a = torch.full((1, T, D), 0.25, dtype=torch.float64, device="cuda")
    a[:, 6000, 3] = 0.0
    gate = (a if form == "linear" else 1 - a).float()
    x = torch.ones(1, T, D, device="cuda")
    x[:, 5, 0], x[:, 40, 1], x[:, 100, 2], x[:, 7, 3] = inf, -inf, float("nan"), inf
    initial = torch.zeros(1, D, device="cuda")
    initial[:, 4] = inf
    d = torch.ones(1, T, D, device="cuda")
    d[:, T - 3, 5], d[:, T - 500, 6], d[:, T - 70, 7] = inf, -inf, float("nan")
    leaves = [v.requires_grad_(True) for v in (gate, x, initial)]
    states, last = gated_scan(*leaves, form=form)
    dx, di = torch.autograd.grad((states, last), leaves[1:], (d, torch.zeros_like(last)))
    want = walk(form, gate.detach().double(), x.detach().double()[:, :, None], initial.detach().double()[:, None], None, False, d.double()[:, :, None], torch.zeros(1, 1, D, dtype=torch.float64, device="cuda"))
    for got, w, what in ((states, want["states"][0][:, :, 0], "states"), (last, want["last"][0][:, 0], "last"), (dx, want["d_x"][0][:, :, 0], "d_x"), (di, want["d_initial"][0][:, 0], "d_initial")):
        for kind in (torch.isnan, torch.isposinf, torch.isneginf):
            assert torch.equal(kind(got), kind(w)), (what, kind.__name__, int((kind(got) != kind(w)).sum()))
        ok = torch.isfinite(w)
        # sums of positive terms that a gate of a quarter forgets: 4 U a step of at most 4 / 3 of the result, and one product
        assert bool(((got.double() - w)[ok].abs() <= 16 * U * w[ok].abs()).all()), what
