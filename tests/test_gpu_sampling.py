"""Draws (gaussian_splatting_amd.sampling, csrc/gsx_draw.hip) against the definition in 64 bits on the host, index for index: a random u lies within
1e-15 of a border between two tokens about once in 1e12 draws, and where borders are met on purpose (equal logits) all sums are whole numbers."""
import math
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def oracle_row(l, u, T, k, p, m):
    """one row, doubles -> (indices, log probabilities)"""
    V = len(l)
    l = np.where(np.isnan(l), -np.inf, l)
    none = np.full(len(u), -1, np.int64), np.full(len(u), -np.inf)
    if V == 0 or not (T >= 0 and p > 0 and 0 <= m <= 1) or l.max() == -np.inf:
        return none
    top = l.max()
    order = sorted(range(V), key=lambda i: (-l[i], i)) if V < 5000 else list(np.argsort(-l, kind="stable"))
    order = np.array(order)
    if T == 0:
        kept, w = order[:1], np.ones(1)
        full = np.zeros(V)
        full[kept] = 1.0
    else:
        with np.errstate(invalid="ignore", over="ignore"):
            w = np.where(l == top, 1.0, np.where(np.isneginf(l) | np.isposinf(top), 0.0, np.exp((l - top) / T)))
        if 0 < k < V:
            order = order[:k]
        if p < 1:
            run = np.cumsum(w[order])
            order = order[:1 + int(np.sum(run < p * run[-1]))]
        order = order[w[order] >= m]
        full = np.zeros(V)
        full[order] = w[order]
    c = np.cumsum(full)
    u = np.where(np.isnan(u), 0.0, np.clip(u, 0.0, 1.0))
    i = np.searchsorted(c, u * c[-1], side="right")
    i = np.minimum(i, np.nonzero(full)[0].max())
    with np.errstate(divide="ignore"):
        return i, np.log(full[i]) - np.log(c[-1])


def check(logits, u, T=1.0, k=0, p=1.0, m=0.0):
    from gaussian_splatting_amd import sample
    R = logits.shape[0]
    f = lambda v, r: float(v[r]) if torch.is_tensor(v) else float(np.float32(v))  # noqa: E731
    got, lp = sample(logits, u, temperature=T, top_k=k, top_p=p, min_p=m, return_logprobs=True)
    assert got.dtype == torch.int64 and got.shape == u.shape and lp.dtype == torch.float32 and lp.shape == u.shape
    assert torch.equal(sample(logits, u, temperature=T, top_k=k, top_p=p, min_p=m), got)
    lh, uh = logits.double().cpu().numpy(), u.double().cpu().numpy()
    got, lp = got.cpu().numpy(), lp.cpu().numpy()
    for r in range(R):
        want, wl = oracle_row(lh[r], uh[r], f(T, r), int(k[r]) if torch.is_tensor(k) else k, f(p, r), f(m, r))
        bad = np.nonzero(got[r] != want)[0]
        assert len(bad) == 0, (r, len(bad), got[r][bad[:4]], want[bad[:4]], uh[r][bad[:4]])
        # one rounding to 32 bits of a difference of 64-bit logarithms
        fin = np.isfinite(wl)
        assert np.array_equal(np.isfinite(lp[r]), fin) and bool((np.abs(lp[r][fin] - wl[fin]) <= 2.0 ** -24 * np.abs(wl[fin]) + 1e-12).all())


def rand(seed, R, V, S, t=torch.float32, sigma=2.0, f64=False):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (sigma * torch.randn(R, V, generator=g, device="cuda")).to(t), torch.rand(R, S, generator=g, device="cuda", dtype=torch.float64 if f64 else torch.float32)


CUTS = [dict(), dict(k=1), dict(k=7, T=0.5), dict(p=0.6), dict(m=0.1, T=1.7), dict(k=40, p=0.9, m=0.02, T=0.8), dict(T=0.0), dict(p=1e-6), dict(p=0.9999), dict(k=1000000), dict(m=1.0)]


@pytest.mark.parametrize("V", [1, 2, 3, 31, 32, 33, 63, 64, 65, 127, 250, 300, 512, 513, 1000, 1025, 4097, 20011])
@pytest.mark.parametrize("cut", CUTS, ids=str)
def test_rows(V, cut):
    dtype = list(DT.values())[V % 3]
    logits, u = rand(V, 5, V, 9, dtype)
    check(logits, u, **cut)


@pytest.mark.parametrize("R,V,S", [(1, 5, 1), (300, 3, 1), (1000, 40, 2), (7, 70001, 33), (2, 200003, 5), (1, 300000, 70000), (600, 1500, 1), (1, 1100003, 100), (130, 40001, 2), (129, 33000, 70), (3, 40000, 300)])
@pytest.mark.parametrize("cut", [dict(), dict(p=0.8), dict(k=300, p=0.95, m=0.001, T=0.9)], ids=str)
def test_sizes(R, V, S, cut):
    logits, u = rand(R + V, R, V, S, sigma=1.5, f64=V > 100000)
    check(logits, u, **cut)


@pytest.mark.parametrize("V", [5, 64, 300, 5000, 100001])
def test_equal_logits_and_borders(V):
    """all sums are whole numbers: every border is met exactly"""
    for value in (0.0, -3.0, torch.finfo(torch.float32).min):
        logits = torch.full((3, V), value, device="cuda")
        grid = torch.arange(0, V + 1, max(1, V // 50), device="cuda", dtype=torch.float64)
        u = (grid / V).clamp(max=1 - 2.0 ** -53).repeat(3, 1)
        exact = torch.floor(u * V)                                    # u * V in doubles, as the definition has it
        from gaussian_splatting_amd import sample
        assert torch.equal(sample(logits, u), exact.long())
        check(logits, u)
        for cut in (dict(k=max(1, V // 3)), dict(p=0.5), dict(p=0.25, k=max(1, V // 2)), dict(m=1.0), dict(T=0.0), dict(p=0.5, m=0.5)):
            check(logits, u, **cut)


def test_more_ties_than_any_list_holds():
    logits = torch.zeros(128, 140000, device="cuda")
    logits[:, ::2] = 1.0
    u = torch.rand(128, 3, device="cuda", generator=torch.Generator(device="cuda").manual_seed(2), dtype=torch.float64)
    check(logits, u, k=100001)
    check(logits[:40], u[:40], p=0.9)


def test_ties_at_the_cut():
    """few values, many times each, in bf16: the last kept ones are the first in index order"""
    g = torch.Generator(device="cuda").manual_seed(4)
    for V in (50, 700, 9000):
        logits = torch.randint(0, 4, (6, V), generator=g, device="cuda").to(torch.bfloat16)
        logits[:, ::7] = -logits[:, ::7]                              # -0 among the zeros
        u = torch.rand(6, 40, generator=g, device="cuda")
        for k in (1, 2, V // 5, V // 3, V - 1):
            check(logits, u, k=k)
            check(logits, u, k=k, p=0.7)
        for p in (0.1, 0.33, 0.5, 0.77, 0.95):
            check(logits, u, p=p)


def test_masked_tokens_and_empty_rows():
    inf, nan, lowest = math.inf, math.nan, torch.finfo(torch.float32).min
    for V in (6, 130, 3000, 70000):
        base, u = rand(V, 8, V, 12)
        base[0] = -inf
        base[1] = nan
        base[2, ::2] = nan
        base[2, 1::2] = -inf
        base[3] = lowest
        base[4, : V // 2] = -inf
        base[4, V // 2] = nan
        base[5, : V - 1] = lowest
        base[6, V // 3] = inf
        base[6, V - 1] = inf
        base[7, 1:] = -inf
        for cut in CUTS:
            check(base, u, **cut)


def test_settings_by_row_and_refused_rows():
    R, V = 10, 900
    logits, u = rand(3, R, V, 6)
    dev = logits.device
    T = torch.tensor([1, 0.5, 0, -1, math.nan, 2, 1, 1, 1, 3.0], device=dev)
    k = torch.tensor([0, 5, 3, 0, 0, -4, 900, 901, 1, 100], dtype=torch.int32, device=dev)
    p = torch.tensor([0.5, 1, 0.9, 0.5, 0.5, 1.5, 0.0, math.nan, 0.7, 0.3], device=dev)
    m = torch.tensor([0, 0.1, 0, 0, 0, 0.01, 0, 0, 2.0, 0.0], device=dev)
    check(logits, u, T=T, k=k, p=p, m=m)
    check(logits, u, T=T)
    check(logits, u, k=k)
    check(logits, u, p=p)
    check(logits, u, m=m)


def test_numbers_at_the_ends():
    for V in (9, 200, 20000):
        logits, _ = rand(1, 2, V, 1)
        logits[:, -1] = -math.inf
        u = torch.tensor([[0.0, -0.5, 1.0, 7.0, math.nan, 1 - 2.0 ** -24, math.inf, -math.inf]] * 2, device="cuda")
        check(logits, u)
        check(logits, u.double(), p=0.5)


def test_extreme_temperatures():
    logits, u = rand(5, 4, 400, 8)
    for T in (1e-30, 1e-4, 1e4, 1e30, 3e38):
        check(logits, u, T=T)
        check(logits, u, T=T, p=0.5)
    check(logits * 1e37, u, T=0.01)
    check(logits * 1e37, u, T=1e36, p=0.9, k=30)


def test_strides_and_types():
    big, u = rand(6, 12, 1003, 4)
    check(big[::3, 5:700], u[::3], p=0.9)
    check(big[:, 1:], u, k=20)
    check(big.t()[:12, :].t()[:, :12], u, m=0.01)                     # tokens that are not consecutive
    check(big.to(torch.bfloat16)[:, 3:], u.double(), p=0.5)
    check(big[:, :640].to(torch.float16)[:, 1:33], u, p=0.5)
    check(big[:1].expand(12, 1003), u, p=0.8)


def test_no_rows_no_tokens_no_draws():
    from gaussian_splatting_amd import sample
    z = lambda *s: torch.zeros(s, device="cuda")  # noqa: E731
    assert sample(z(0, 5), z(0, 3)).shape == (0, 3)
    assert sample(z(4, 5), z(4, 0)).shape == (4, 0)
    i, lp = sample(z(4, 0), z(4, 3), top_k=3, top_p=0.5, return_logprobs=True)
    assert bool((i == -1).all()) and bool((lp == -math.inf).all())


def test_many_short_rows():
    g = torch.Generator(device="cuda").manual_seed(8)
    for V in (2, 17, 32, 48, 100):
        logits = torch.log(torch.rand(3000, V, generator=g, device="cuda"))
        logits[torch.rand(3000, V, generator=g, device="cuda") < 0.5] = -math.inf
        u = torch.rand(3000, 3, generator=g, device="cuda")
        check(logits, u, m=0.01)
        check(logits[:500], u[:500], p=0.9, k=3)


def test_the_same_bits_on_another_stream_and_when_replayed():
    from gaussian_splatting_amd import sample
    shapes = [(3, 50000, 4), (200, 30, 2), (1, 400000, 5000), (300, 2000, 1)]
    sets = [rand(n, R, V, S) for n, (R, V, S) in enumerate(shapes)]
    work = lambda: [sample(l, u, temperature=0.8, top_k=5000, top_p=0.9, min_p=1e-4, return_logprobs=True) for l, u in sets]  # noqa: E731
    flat = lambda r: [t.clone() for pair in r for t in pair]  # noqa: E731
    first = flat(work())
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        second = flat(work())
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(first, second))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = work()
    for n in range(4):
        for l, u in sets:
            l.copy_(2 * torch.randn(l.shape, device="cuda"))
            u.copy_(torch.rand(u.shape, device="cuda"))
        graph.replay()
        torch.cuda.synchronize()
        got = flat(out)
        assert all(torch.equal(a, b) for a, b in zip(got, flat(work()))), n


def test_dense_points():
    from gaussian_splatting_amd import GaussianSplat
    torch.manual_seed(3)
    m = GaussianSplat(5000).cuda()
    u = torch.rand(2000, device="cuda", dtype=torch.float64)
    pts = m.get_dense_points(2000, temperature=0.1, top_p=0.8, uniforms=u)
    want, _ = oracle_row(m.opacity.detach().double().cpu().numpy()[:, 0], u.cpu().numpy(), float(np.float32(0.1)), 0, float(np.float32(0.8)), 0.0)
    want = torch.from_numpy(want).cuda()
    assert torch.equal(pts, torch.cat([m.positions[want], m.features[want]], 1))
    assert m.get_dense_points(100, min_p=0.5).shape == (100, 6) and m.get_dense_points(0, min_p=0.5).shape == (0, 6)
    # without any of the new arguments: the draws that it made before
    torch.manual_seed(7)
    a = m.get_dense_points(300)
    torch.manual_seed(7)
    i = torch.multinomial(torch.softmax(m.opacity.detach().squeeze(-1), 0), 300, replacement=True)
    assert torch.equal(a, torch.cat([m.positions[i], m.features[i]], 1))
    with torch.no_grad():
        m.opacity.fill_(math.nan)
    with pytest.raises(ValueError, match="no Gaussian is left"):
        m.get_dense_points(10, top_k=5)


def test_ranks_by_row_beyond_32_bits():
    logits, u = rand(11, 4, 700, 6)
    k = torch.tensor([2 ** 33, 2 ** 32 + 5, 3, -(2 ** 40)], device="cuda")
    check(logits, u, k=k)


@pytest.mark.parametrize("R,V,S,t", [(3, 600001, 40, "bf16"), (2, 90000, 40000, "f16"), (5, 70000, 9, "bf16"), (1, 9000011, 40000, "f32")])
def test_rows_in_parts_with_settings_by_row(R, V, S, t):
    """more than one part, walker and node, every type, many draws of several rows"""
    logits, u = rand(R + S, R, V, S, DT[t], f64=True)
    check(logits, u)
    dev = logits.device
    by_row = dict(T=torch.linspace(0.5, 1.1, R, device=dev), k=torch.arange(R, device=dev) * 700, p=torch.linspace(0.99, 0.4, R, device=dev), m=torch.linspace(0, 0.001, R, device=dev))
    check(logits, u, **by_row)
    if R > 1:
        logits[0, ::3], logits[1, : V - 1] = math.inf, -math.inf
        check(logits, u, p=0.5)


@pytest.mark.parametrize("R,V", [(11000, 200000), (4000, 600000)])
def test_offsets_beyond_32_bits(R, V):
    """rows that begin behind 2^31 elements: the same draws as the rows by themselves"""
    from gaussian_splatting_amd import sample
    logits = torch.empty(R, V, dtype=torch.bfloat16, device="cuda")
    logits[: R - 3] = 0
    logits[R - 3:], u = rand(12, 3, V, 4, torch.bfloat16, f64=True)
    us = torch.zeros(R, 4, dtype=torch.float64, device="cuda")
    us[R - 3:] = u
    for cut in (dict(), dict(k=500, p=0.9)):
        got = sample(logits, us, top_k=cut.get("k", 0), top_p=cut.get("p", 1.0))
        assert bool((got[: R - 3] == 0).all())
        check(logits[R - 3:], u, **cut)
        assert torch.equal(got[R - 3:], sample(logits[R - 3:], u, top_k=cut.get("k", 0), top_p=cut.get("p", 1.0)))


def test_two_streams_at_once():
    from gaussian_splatting_amd import sample
    sets = [rand(20 + n, R, V, S, f64=True) for n, (R, V, S) in enumerate([(2, 300000, 50), (200, 9000, 3), (2000, 40, 2)])]
    alone = [sample(l, u, top_p=0.9) for l, u in sets]
    streams = [torch.cuda.Stream() for _ in sets]
    torch.cuda.synchronize()
    outs = [[] for _ in sets]
    for _ in range(5):
        for s, (l, u), o in zip(streams, sets, outs):
            with torch.cuda.stream(s):
                o.append(sample(l, u, top_p=0.9))
    torch.cuda.synchronize()
    assert all(torch.equal(a, o) for a, out in zip(alone, outs) for o in out)


def test_in_inference_mode():
    from gaussian_splatting_amd import sample, gated_scan, gated_step
    with torch.inference_mode():
        logits, u = rand(30, 3, 1000, 5)
        check(logits, u, k=20)
        state, z, x = torch.zeros(3, 1000, device="cuda"), torch.rand(3, 1000, device="cuda"), torch.randn(3, 1000, device="cuda")
        _, last = gated_scan(z[:, None], x[:, None])
        assert torch.equal(gated_step(state, z, x), last)


def test_the_longest_row():
    from gaussian_splatting_amd import sample
    from gaussian_splatting_amd.sampling import MAX_V
    u = torch.rand(1, 300, device="cuda", dtype=torch.float64, generator=torch.Generator(device="cuda").manual_seed(41))
    logits = torch.zeros(1, MAX_V, device="cuda")
    assert torch.equal(sample(logits, u), torch.floor(u * MAX_V).long())                 # whole numbers: exact
    assert torch.equal(sample(logits, u, top_k=MAX_V // 2), torch.floor(u * (MAX_V // 2)).long())
    logits.normal_(generator=torch.Generator(device="cuda").manual_seed(42))
    w = torch.exp(logits[0].double() - logits.max().double())
    rank = torch.sort(logits[0], descending=True, stable=True).indices
    run = torch.cumsum(w[rank], 0)
    keep = 1 + int((run < float(np.float32(0.7)) * run[-1]).sum())
    kept = torch.zeros_like(w)
    kept[rank[:keep]] = w[rank[:keep]]
    c = torch.cumsum(kept, 0)
    assert torch.equal(sample(logits, u, top_p=0.7)[0], torch.searchsorted(c, u[0] * c[-1], right=True))
    with pytest.raises(ValueError, match="tokens"):
        sample(torch.zeros(1, 1, device="cuda").expand(1, MAX_V + 1), u)


@pytest.mark.parametrize("R,V,S", [(300, 20001, 2), (260, 65536, 17), (260, 66000, 3), (300, 17000, 30), (3, 49152, 65), (2, 49153, 20), (257, 600, 16)])
@pytest.mark.parametrize("cut", [dict(), dict(k=300, p=0.95, T=0.9), dict(p=0.7, T=30.0)], ids=str)
def test_more_rows_than_compute_units(R, V, S, cut):
    """both sides of the choices by the number of rows; the high temperature leaves more tokens in a bin than are ranked at once"""
    from gaussian_splatting_amd import sample
    logits, u = rand(R + V + S, R, V, S, f64=True)
    rows = [0, 1, R // 2, R - 1]
    got = sample(logits, u, temperature=cut.get("T", 1.0), top_k=cut.get("k", 0), top_p=cut.get("p", 1.0)).cpu().numpy()
    for r in rows:
        want, _ = oracle_row(logits[r].double().cpu().numpy(), u[r].cpu().numpy(), float(np.float32(cut.get("T", 1.0))), cut.get("k", 0), float(np.float32(cut.get("p", 1.0))), 0.0)
        assert np.array_equal(got[r], want), (r, got[r], want)


@pytest.mark.parametrize("S", [8192, 8193, 30000])
@pytest.mark.parametrize("cut", [dict(k=100), dict(k=161, p=0.6, m=0.07, T=0.35)], ids=str)
def test_many_draws_from_few_tokens(S, cut):
    logits, u = rand(S, 2, 100001, S, f64=True)
    check(logits, u, **cut)


NEAR_ONE = [1.0, 1 - 2.0 ** -53, 7.0, math.inf, 1 - 2.0 ** -52, 1 - 2.0 ** -50, 0.5]


@pytest.mark.parametrize("R,V,S", [(2, 15000, 7), (2, 15000, 70), (130, 70000, 7), (130, 70000, 18), (2, 300000, 7), (1, 1100003, 40000)])
@pytest.mark.parametrize("cut", [dict(k=700), dict(m=0.01)], ids=str)
def test_numbers_of_one_where_the_kept_tokens_come_first(R, V, S, cut):
    """a thread or a wave of the row (both sizes), of the pick kernel, of the parts: behind the last kept token all sums agree but for rounding"""
    from gaussian_splatting_amd import sample
    g = torch.Generator(device="cuda").manual_seed(V + S)
    logits = torch.full((R, V), -30.0, device="cuda")
    logits[:, :700] = torch.rand(R, 700, generator=g, device="cuda")
    u = torch.rand(R, S, generator=g, device="cuda", dtype=torch.float64)
    u[:, :7] = torch.tensor(NEAR_ONE, dtype=torch.float64, device="cuda")
    got = sample(logits, u, top_k=cut.get("k", 0), min_p=cut.get("m", 0.0)).cpu().numpy()
    for r in {0, R - 1}:
        want, _ = oracle_row(logits[r].double().cpu().numpy(), u[r].cpu().numpy(), 1.0, cut.get("k", 0), 1.0, float(np.float32(cut.get("m", 0.0))))
        assert want[0] == 699 and np.array_equal(got[r], want), (r, np.nonzero(got[r] != want)[0][:5])
    u32 = u.float()
    assert torch.equal(sample(logits, u32, top_k=cut.get("k", 0), min_p=cut.get("m", 0.0))[:, :4], torch.from_numpy(got[:, :4]).cuda())


def test_a_number_of_one_and_the_longest_row():
    """the kept tokens are the first of 2^27: the draw looks for the last of them, it does not walk there (33 million groups, seconds)"""
    from gaussian_splatting_amd import sample
    from gaussian_splatting_amd.sampling import MAX_V
    logits = torch.full((1, MAX_V), -100.0, dtype=torch.bfloat16, device="cuda")
    logits[:, :600] = 1.0
    u = torch.tensor([[1.0, 1 - 2.0 ** -53, 0.5, 2.0]], dtype=torch.float64, device="cuda")
    sample(logits, u * 0.5, top_k=600)
    start, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    start.record()
    got = sample(logits, u, top_k=600)
    end.record()
    assert got.tolist() == [[599, 599, 300, 599]]
    assert start.elapsed_time(end) < 500.0                            # ms: a few for the passes


def test_more_rows_and_draws_than_one_axis_of_a_launch():
    """more than 2^32 threads in each kind of kernel: lanes of short rows, workgroups of rows, threads of draws"""
    from gaussian_splatting_amd import sample
    g = torch.Generator(device="cuda").manual_seed(5)
    for R, V in (((1 << 26) + 5, 200), ((1 << 23) + 3, 513)):
        logits = 2 * torch.randn(1, V, generator=g, device="cuda")
        u = torch.rand(R, 1, generator=g, device="cuda", dtype=torch.float64)
        c = torch.cumsum(torch.exp(logits[0].double() - logits.max().double()), 0)
        got = sample(logits.expand(R, V), u)
        for r in range(0, R, 1 << 24):
            want = torch.searchsorted(c, u[r:r + (1 << 24), 0] * c[-1], right=True)
            assert torch.equal(got[r:r + (1 << 24), 0], want), (R, V, r)
        del got, u
    R, V = 600, 700
    S = (1 << 32) // R + 9
    logits = 2 * torch.randn(1, V, generator=g, device="cuda")
    u = torch.rand(1, S, generator=g, device="cuda")
    c = torch.cumsum(torch.exp(logits[0].double() - logits.max().double()), 0)
    want = torch.searchsorted(c, u[0].double() * c[-1], right=True)
    got = sample(logits.expand(R, V), u.expand(R, S))
    for r in range(R):
        assert torch.equal(got[r], want), r


@pytest.mark.parametrize("R,V,S", [(1, 2, 100003), (1, 7, 1025), (1, 300, 250000), (1, 512, 100000), (3, 30, 40001), (33, 100, 4099), (70, 5, 3000), (1030, 30, 1300)])
@pytest.mark.parametrize("cut", [dict(), dict(k=5, p=0.7, m=0.01, T=0.8)], ids=str)
def test_many_draws_from_short_rows(R, V, S, cut):
    """a wave's draws in shares: rows that meet within a share, shares that end within a row, the last of each"""
    logits, u = rand(R + V + S, R, V, S, DT[list(DT)[V % 3]], f64=True)
    check(logits, u, **cut)


def test_dense_points_of_a_small_scene():
    from gaussian_splatting_amd import GaussianSplat
    torch.manual_seed(4)
    m = GaussianSplat(300).cuda()
    u = torch.rand(1000000, device="cuda", dtype=torch.float64)
    m.get_dense_points(1000000, top_p=0.9, uniforms=u)
    start, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    start.record()
    pts = m.get_dense_points(1000000, top_p=0.9, uniforms=u)
    end.record()
    end.synchronize()
    assert start.elapsed_time(end) < 6.0                              # ms: one wave alone takes 12
    want, _ = oracle_row(m.opacity.detach().double().cpu().numpy()[:, 0], u.cpu().numpy(), 1.0, 0, float(np.float32(0.9)), 0.0)
    want = torch.from_numpy(want).cuda()
    assert torch.equal(pts, torch.cat([m.positions[want], m.features[want]], 1))


@pytest.mark.parametrize("R,V", [(4100, 524301), (128, 200001)])
def test_lists_that_do_not_fit(R, V):
    """many long rows, whose cuts lie among more tokens than the row's list has room for (4096, and 131072)"""
    from gaussian_splatting_amd import sample
    g = torch.Generator(device="cuda").manual_seed(R)
    logits = torch.randn(R, V, generator=g, device="cuda", dtype=torch.bfloat16)
    u = torch.rand(R, 5, generator=g, device="cuda", dtype=torch.float64)
    for cut in (dict(T=300.0, p=0.6), dict(T=300.0, k=V // 2, p=0.9)):
        got = sample(logits, u, temperature=cut["T"], top_k=cut.get("k", 0), top_p=cut["p"]).cpu().numpy()
        for r in (0, R // 3, R - 1):
            want, _ = oracle_row(logits[r].double().cpu().numpy(), u[r].cpu().numpy(), 300.0, cut.get("k", 0), float(np.float32(cut["p"])), 0.0)
            assert np.array_equal(got[r], want), (r, cut, got[r], want)


@pytest.mark.parametrize("R,V,S", [(2, 3001, 5), (2, 3001, 70), (300, 40001, 5), (2, 40001, 5), (2, 40001, 70), (129, 120001, 3), (2, 100001, 5), (2, 100001, 40000), (128, 300001, 3)])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_long_ties_under_both_cuts(R, V, S, dtype):
    """top-k and top-p together among more equal tokens than are ranked at once, through every kernel that finds a cut exactly: the row's own of 512 threads (3001,
    300 x 40001), the one behind the row's of 1024 (2 x 40001, 129 x 120001), the one of rows in parts, from its list and (300001) from the row"""
    from gaussian_splatting_amd import sample
    g = torch.Generator(device="cuda").manual_seed(V)
    logits = torch.randint(0, 2, (R, V), generator=g, device="cuda").to(DT[dtype])
    u = torch.rand(R, S, generator=g, device="cuda", dtype=torch.float64)
    rows = sorted({0, 1, R // 2, R - 1})
    for k, p, m in ((V // 3, 0.5, 0.0), (V - V // 4, 0.8, 0.0), (V - 1, 0.97, 0.0), (2 * V // 3, 0.6, 0.5), (700, 0.9, 0.0)):
        got = sample(logits, u, top_k=k, top_p=p, min_p=m).cpu().numpy()
        for r in rows:
            want, _ = oracle_row(logits[r].double().cpu().numpy(), u[r].cpu().numpy(), 1.0, k, float(np.float32(p)), float(np.float32(m)))
            assert np.array_equal(got[r], want), (r, k, p, np.nonzero(got[r] != want)[0][:4])


@pytest.mark.parametrize("t,k", [(torch.uint64, [2 ** 32 + 3, 3, 0, 700]), (torch.uint32, [2 ** 31 + 5, 2 ** 32 - 1, 4, 0]), (torch.uint16, [65535, 2, 0, 100]), (torch.uint8, [255, 1, 0, 7])], ids=str)
def test_ranks_by_row_of_unsigned_types(t, k):
    from gaussian_splatting_amd import sample
    logits, u = rand(13, 4, 700, 50)
    want = torch.tensor([min(v, 700) for v in k], dtype=torch.int32, device="cuda")
    assert torch.equal(sample(logits, u, top_k=torch.tensor(k, dtype=t).cuda()), sample(logits, u, top_k=want))


@pytest.mark.parametrize("V", [6, 300, 5000, 17001, 70000])
def test_settings_near_zero(V):
    """a temperature that 32 bits round to 0 still shares the draws out among equal largest logits, and such a share still keeps the first token"""
    from gaussian_splatting_amd import sample
    logits, u = rand(V, 2, V, 400, f64=True)
    ties = torch.tensor([1, V // 2, V - 2], device="cuda")
    logits[:, ties] = 20.0
    want = ties[(u * 3).floor().long()]
    R = torch.full((2,), 1.0, dtype=torch.float64, device="cuda")
    for T in (1e-50, 5e-324, 2.0 ** -149, 1e-40, 1e-37):
        assert torch.equal(sample(logits, u, temperature=T), want), T
        assert torch.equal(sample(logits, u, temperature=R * T), want), T
        assert torch.equal(sample(logits, u, temperature=T, top_p=0.5), ties[(u * 2).floor().long()]), T
        assert torch.equal(sample(logits, u, temperature=T, top_k=2), ties[(u * 2).floor().long()]), T
    for p in (1e-50, 5e-324, 2.0 ** -149, 1e-40):
        assert bool((sample(logits, u, top_p=p) == 1).all()) and bool((sample(logits, u, top_p=R * p) == 1).all()), p
    assert bool((sample(logits, u, temperature=0.0) == 1).all()) and bool((sample(logits, u, temperature=R * 0) == 1).all()) and bool((sample(logits, u, top_p=R * 0) == -1).all())
