"""CPU tier of the gated scan and the draws: what is refused, before any GPU is touched."""
import ctypes as C
import math
import pytest
import torch
from gaussian_splatting_amd import GaussianSplat, composite_layers, gated_scan, gated_step, sample
from gaussian_splatting_amd import _lib as L


def z(*s, t=torch.float32):
    return torch.zeros(s, dtype=t)


def test_scan_refusals():
    x = z(2, 5, 3)
    for gate, xx, kw, err, match in [
        (x, x, dict(), RuntimeError, "no CPU fallback"),
        (x, z(2, 5, 4), dict(), ValueError, "wanted"),
        (z(2, 5), z(2, 5), dict(), ValueError, "wanted"),
        (x, z(2, 5, 5, 3), dict(), ValueError, "planes"),
        (x, z(2, 5, 0, 3), dict(), ValueError, "planes"),
        (x, z(2, 5, 3, t=torch.float16), dict(), TypeError, "share"),
        (x.double(), x.double(), dict(), TypeError, "share"),
        (x, x, dict(form="lstm"), ValueError, "form"),
        (x, x, dict(initial=z(2, 4)), ValueError, "initial"),
        (x, x, dict(initial=z(2, 3, t=torch.int32)), ValueError, "initial"),
        (x, x, dict(lengths=z(2, t=torch.int64)), ValueError, "lengths"),
        (x, x, dict(lengths=z(3, t=torch.int32)), ValueError, "lengths"),
    ]:
        with pytest.raises(err, match=match):
            gated_scan(gate, xx, **kw)


def test_step_refusals():
    for state, gate, x, err, match in [
        (z(4), z(4), z(4), RuntimeError, "no CPU fallback"),
        (z(4, t=torch.bfloat16), z(4), z(4), ValueError, "state"),
        (z(4), z(5), z(4), ValueError, "share"),
        (z(4, 6).t(), z(6, 4), z(6, 4), ValueError, "contiguous"),
        (z(4), z(4, t=torch.float16), z(4), TypeError, "share"),
    ]:
        with pytest.raises(err, match=match):
            gated_step(state, gate, x)


def test_layers_refusals():
    rgb, alpha = z(3, 2, 3, 4, 5), z(3, 2, 1, 4, 5)
    for args, err, match in [((rgb, alpha), RuntimeError, "no CPU fallback"), ((rgb, z(3, 2, 3, 4, 5)), ValueError, "wanted"), ((rgb[0], alpha[0]), ValueError, "wanted"),
                             ((z(3, 2, 5, 4, 5), alpha), ValueError, "planes"), ((rgb, alpha, z(3, 4, 5)), ValueError, "background")]:
        with pytest.raises(err, match=match):
            composite_layers(*args)


def test_draw_refusals():
    l, u = z(2, 7), z(2, 3)
    for args, kw, err, match in [
        ((l, u), dict(), RuntimeError, "no CPU fallback"),
        ((l, z(3, 3)), dict(), ValueError, "wanted"),
        ((l[0], u[0]), dict(), ValueError, "wanted"),
        ((l.double(), u), dict(), TypeError, "logits"),
        ((l, u.half()), dict(), TypeError, "uniforms"),
        ((l, u), dict(temperature=-1.0), ValueError, "temperature"),
        ((l, u), dict(temperature=math.nan), ValueError, "temperature"),
        ((l, u), dict(top_k=-1), ValueError, "top_k"),
        ((l, u), dict(top_k=1.5), ValueError, "top_k"),
        ((l, u), dict(top_p=0.0), ValueError, "top_p"),
        ((l, u), dict(min_p=1.5), ValueError, "min_p"),
        ((l, u), dict(min_p=math.nan), ValueError, "min_p"),
        ((l, u), dict(top_p=z(3)), ValueError, "top_p"),
        ((z(1, 1).expand(1, (1 << 27) + 1), z(1, 1)), dict(), ValueError, "tokens"),
    ]:
        with pytest.raises(err, match=match):
            sample(*args, **kw)
    m = GaussianSplat(6)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        m.get_dense_points(5, top_k=2)
    with pytest.raises(ValueError, match="one uniform"):
        m.get_dense_points(5, uniforms=z(4))
    with pytest.raises(ValueError, match="one logit"):
        m.get_dense_points(5, logits=z(4))


def test_ranks_by_row_are_whole_numbers():
    from gaussian_splatting_amd import sample
    with pytest.raises(TypeError, match="whole numbers"):
        sample(torch.zeros(3, 5), torch.zeros(3, 2), top_k=torch.full((3,), 2.5))


def test_c_entry_points_refuse_before_the_device():
    lib = L.lib()
    ok = dict(dtype=0, form=0, planes=1, B=1, T=2, D=3)
    gated = lambda **kw: L.GsxGated(**dict(ok, **kw))  # noqa: E731
    for fn in (lib.gsx_gated_scan_fwd, lib.gsx_gated_scan_bwd):
        assert fn(None, None) == L.GSX_E_INVALID
        for bad in (dict(dtype=3), dict(form=-1), dict(form=3), dict(planes=0), dict(planes=5), dict(B=-1), dict(T=-1), dict(D=-1), dict()):
            assert fn(gated(**bad), None) == L.GSX_E_INVALID, bad
        assert fn(gated(D=1 << 31), None) == L.GSX_E_RANGE
        assert fn(gated(B=1 << 30, D=1 << 30), None) == L.GSX_E_RANGE
        assert fn(gated(B=0), None) == L.GSX_OK and fn(gated(D=0), None) == L.GSX_OK
    assert lib.gsx_gated_marks_floats(1, -1, 1, 1) == L.GSX_E_INVALID and lib.gsx_gated_marks_floats(1, 1, 5, 1) == L.GSX_E_INVALID
    assert lib.gsx_gated_marks_floats(2, 0, 1, 9) == 0 and lib.gsx_gated_marks_floats(2, 1, 3, 9) == 54
    assert lib.gsx_gated_step(0, 0, 4, None, None, None, None) == L.GSX_E_INVALID
    assert lib.gsx_gated_step(0, 0, 0, None, None, None, None) == L.GSX_OK
    assert lib.gsx_gated_step(0, 0, -1, None, None, None, None) == L.GSX_E_INVALID
    assert lib.gsx_gated_step(5, 0, 1, None, None, None, None) == L.GSX_E_INVALID
    ok = dict(dtype=0, R=2, V=10, S=1, row_stride=10, temperature=1.0, top_p=1.0, min_p=0.0, top_k=0)
    draw = lambda **kw: L.GsxDraw(**dict(ok, **kw))  # noqa: E731
    assert lib.gsx_draw_indices(None, None) == L.GSX_E_INVALID and lib.gsx_draw_workspace_bytes(None) == 0
    for bad in (dict(dtype=9), dict(R=-1), dict(V=-1), dict(S=-1), dict(temperature=-1.0), dict(temperature=math.nan), dict(top_p=0.0), dict(min_p=-0.1), dict(min_p=1.1), dict(top_k=-1)):
        assert lib.gsx_draw_indices(draw(**bad), None) == L.GSX_E_INVALID and lib.gsx_draw_workspace_bytes(draw(**bad)) == 0, bad
    assert lib.gsx_draw_indices(draw(), None) == L.GSX_E_INVALID                    # null pointers
    assert lib.gsx_draw_indices(draw(V=(1 << 27) + 1), None) == L.GSX_E_RANGE and lib.gsx_draw_indices(draw(R=1 << 31), None) == L.GSX_E_RANGE
    assert lib.gsx_draw_indices(draw(R=0), None) == L.GSX_OK and lib.gsx_draw_indices(draw(S=0), None) == L.GSX_OK
    s = draw(logits=4096, uniforms=4096, indices=4096, ws=4096, ws_bytes=1)
    assert lib.gsx_draw_workspace_bytes(draw()) > 1 and lib.gsx_draw_indices(s, None) == L.GSX_E_CAPACITY
    s = draw(logits=4096, uniforms=4096, indices=4096, ws=4100, ws_bytes=1 << 20)
    assert lib.gsx_draw_indices(s, None) == L.GSX_E_INVALID                         # a workspace off its boundary


def test_structs_match_the_header():
    """the library's own view of the two structs: a size that disagreed would shift every field behind it"""
    import os
    import subprocess
    import tempfile
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    src = '#include <stdio.h>\n#include "gsx.h"\nint main(void) { printf("%zu %zu %zu %zu\\n", sizeof(gsx_gated), offsetof(gsx_gated, d_initial), sizeof(gsx_draw), offsetof(gsx_draw, ws_bytes)); return 0; }\n'
    with tempfile.TemporaryDirectory() as d:
        open(os.path.join(d, "a.c"), "w").write(src)
        subprocess.check_call(["gcc", "-I", os.path.join(root, "include"), os.path.join(d, "a.c"), "-o", os.path.join(d, "a")])
        got = [int(v) for v in subprocess.check_output([os.path.join(d, "a")], text=True).split()]
    assert got == [C.sizeof(L.GsxGated), L.GsxGated.d_initial.offset, C.sizeof(L.GsxDraw), L.GsxDraw.ws_bytes.offset]


@pytest.mark.parametrize("V", [0, 10, 512, 513, 49152, 49153, 60000, 524284, 524285, 1 << 27])
def test_workspace_of_a_batch_without_rows_or_draws(V):
    """what a C caller asks for before a call that does nothing: a size, for every way that V alone would take"""
    lib = L.lib()
    for cut in (dict(), dict(top_k=5, top_p=0.5)):
        s = dict(dtype=0, R=2, V=V, S=1, row_stride=V, temperature=1.0, top_p=1.0, min_p=0.0, top_k=0)
        for none in (dict(R=0), dict(S=0), dict(R=0, S=0)):
            d = L.GsxDraw(**dict(s, **cut, **none))
            assert 0 < lib.gsx_draw_workspace_bytes(d) <= 256 and lib.gsx_draw_indices(d, None) == L.GSX_OK


def test_first_calls_of_two_threads(monkeypatch):
    """a second thread that comes while the first one fills the table of entry points gets a whole table"""
    import threading
    from gaussian_splatting_amd import recurrence
    real, seen, threads = L.lib(), [], []

    class Slow:
        def __getitem__(self, name):
            if name == "gsx_gated_scan_bwd" and not threads:         # two of the three are in the first thread's hands
                threads.append(threading.Thread(target=lambda: seen.append(set(recurrence._entries()))))
                threads[0].start()
                threads[0].join()
            return real[name]
    slow = Slow()
    monkeypatch.setattr(L, "lib", lambda: slow)
    monkeypatch.setattr(recurrence, "_entry", None)
    want = {"gsx_gated_workspace_bytes", "gsx_gated_scan_fwd", "gsx_gated_scan_bwd"}
    assert set(recurrence._entries()) == want and seen == [want]


@pytest.mark.parametrize("k,err", [(math.inf, ValueError), (-math.inf, ValueError), (math.nan, ValueError)])
def test_ranks_that_are_no_numbers_of_tokens(k, err):
    """an endless rank is no whole number"""
    with pytest.raises(err, match="top_k"):
        sample(z(3, 5), z(3, 2), top_k=k)


def test_marks_beyond_64_bits_are_refused():
    """inputs with strides of zero need no memory, so the size is the only thing that stands in the way of such a call"""
    size = L.lib().gsx_gated_marks_floats
    for args in ((1, 1 << 39, 1, 1 << 30), (1 << 20, (1 << 40) - 16, 4, 1 << 20), (1 << 20, 1 << 30, 1, 1 << 20), (1 << 31, 1, 1, 1), (1, 1 << 40, 1, 1), (1, 1, 1, 1 << 31), (1 << 21, 1, 1, 1 << 20)):
        assert size(*args) == L.GSX_E_RANGE, args
    assert size(1, (1 << 40) - 1, 1, 1) == 1 << 36 and size(1 << 20, 16, 1, 1 << 20) == 1 << 40 and size(0, 1 << 30, 4, 1 << 30) == 0


@pytest.mark.parametrize("which", [0, 1, 2], ids=["state", "gate", "x"])
def test_step_refuses_to_drop_a_gradient(which):
    args = [z(4), z(4), z(4)]
    args[which].requires_grad_(True)
    with pytest.raises(RuntimeError, match="require a gradient"):
        gated_step(*args)
    with torch.no_grad(), pytest.raises(RuntimeError, match="no CPU fallback"):
        gated_step(*args)


def test_step_refuses_inputs_that_overlap_the_state():
    """addresses only: none of these calls reaches a device"""
    lib, at, n = L.lib(), 1 << 20, 64
    far = at + 4096
    for dtype, size in ((0, 4), (1, 2), (2, 2)):
        for other in (at + 4, at - 4, at + 4 * n - size, at - size * n + size) + ((at,) if size == 2 else ()):
            assert lib.gsx_gated_step(dtype, 0, n, at, other, far, None) == L.GSX_E_INVALID, (dtype, other - at)
            assert lib.gsx_gated_step(dtype, 0, n, at, far, other, None) == L.GSX_E_INVALID, (dtype, other - at)


def test_what_is_packed_is_the_struct(monkeypatch):
    """both directions of a scan up to the library's door, which is replaced: every field of the struct holds what it is named for"""
    from gaussian_splatting_amd import recurrence
    calls = []

    def door(name):
        def entry(packed, other):
            assert len(packed) == C.sizeof(L.GsxGated)
            calls.append((name, L.GsxGated.from_buffer_copy(packed)))
            return 512 if name.endswith("bytes") else 0
        return entry
    monkeypatch.setattr(recurrence, "_entry", {n: door(n) for n in ("gsx_gated_workspace_bytes", "gsx_gated_scan_fwd", "gsx_gated_scan_bwd")})
    monkeypatch.setattr(recurrence, "_refuse_host", lambda x, name: None)
    monkeypatch.setattr(L, "stream_ptr", lambda dev: 0)
    B, T, P, D = 2, 5, 3, 7
    gate, x = z(T, B, D + 1, t=torch.bfloat16)[:, :, 1:].transpose(0, 1), z(B, T, P, D, t=torch.bfloat16)
    initial, lengths = z(B, P, D), torch.tensor([3, 5], dtype=torch.int32)
    leaves = [v.requires_grad_(True) for v in (gate, x, initial)]
    states, last = gated_scan(*leaves, lengths=lengths, form="over", reverse=True)
    grads = torch.autograd.grad((states, last), leaves, (z(B, T, P, D, t=torch.bfloat16), z(B, P, D)))
    assert [n for n, _ in calls] == ["gsx_gated_workspace_bytes", "gsx_gated_scan_fwd", "gsx_gated_workspace_bytes", "gsx_gated_scan_bwd"]
    (_, sized), (_, f), _, (_, b) = calls
    assert sized.ws is None and sized.ws_bytes == 0
    for s in (f, b):
        assert (s.dtype, s.form, s.reverse, s.planes, s.B, s.T, s.D) == (1, 2, 1, P, B, T, D)
        assert s.gate == gate.data_ptr() and list(s.gate_stride) == [D + 1, B * (D + 1)] and s.x == x.data_ptr() and list(s.x_stride) == [T * P * D, P * D, D]
        assert s.lengths == lengths.data_ptr() and s.marks and s.ws and s.ws_bytes == 512
    assert f.initial == initial.data_ptr() and f.states == states.data_ptr() and f.last == last.data_ptr() and f.marks == b.marks
    assert not (f.d_states or f.d_last or f.d_gate or f.d_x or f.d_initial or b.initial or b.states or b.last)
    assert b.d_states and list(b.d_states_stride) == [T * P * D, P * D, D] and b.d_last
    assert [b.d_gate, b.d_x, b.d_initial] == [g.data_ptr() for g in grads]
