"""The gated linear recurrence h_t = a_t h_(t-1) + b_t along one axis as one HIP pass each way (csrc/gsx_gated.hip): the formula by
which depth-ordered splats are composited (/root/reference/model/gaussian_splatting.py:143-144), by itself -- for layers
(render.composite_layers), for decayed traces of per-Gaussian scores over views, for gated sequence models.

    linear   h_t = z_t h_(t-1) + x_t
    blend    h_t = (1 - z_t) h_(t-1) + z_t x_t          (straight colours over each other, z = alpha)
    over     h_t = (1 - z_t) h_(t-1) + x_t              (premultiplied colours)"""
import torch
from . import _lib as L

FORMS = {"linear": 0, "blend": 1, "over": 2}                     # GSX_GATED_*
DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}   # GSX_F32, GSX_BF16, GSX_F16
MAX_PLANES = 4                                                   # GSX_GATED_MAX_PLANES


def _ptr(t):
    return t.data_ptr() if t is not None else None


def _channels(t):
    """t with its channels one element apart (every other stride is the kernel's business)"""
    return t if t.shape[-1] <= 1 or t.stride(-1) == 1 else t.contiguous()


def _shape(gate, x, lengths, form, reverse):
    s = L.GsxGated()
    s.dtype = DTYPES[x.dtype]; s.form = FORMS[form]; s.reverse = int(reverse)
    s.B, s.T, s.D = gate.shape
    s.planes = x.shape[2] if x.dim() == 4 else 1
    s.gate = _ptr(gate); s.gate_stride[:] = [gate.stride(0), gate.stride(1)]
    s.x = _ptr(x); s.x_stride[:] = [x.stride(0), x.stride(1), x.stride(2) if x.dim() == 4 else 0]
    s.lengths = _ptr(lengths)
    return s


def _workspace(lib, s, backward, dev):
    n = lib.gsx_gated_workspace_bytes(s, backward)
    if not n:
        return None
    ws = torch.empty(n, dtype=torch.uint8, device=dev)
    s.ws = _ptr(ws); s.ws_bytes = n
    return ws


class _GatedScan(torch.autograd.Function):
    @staticmethod
    def forward(ctx, gate, x, initial, lengths, form, reverse, want_states, want_grad):
        lib = L.lib()
        gate, x = _channels(gate.detach()), _channels(x.detach())
        dev = x.device
        state_shape = x.shape[:1] + x.shape[2:]
        h0 = initial.detach().to(torch.float32).contiguous() if initial is not None else None
        states = torch.empty(x.shape, dtype=x.dtype, device=dev) if want_states else None
        last = torch.empty(state_shape, dtype=torch.float32, device=dev)
        s = _shape(gate, x, lengths, form, reverse)
        marks = None
        if want_grad:
            marks = torch.empty(lib.gsx_gated_marks_floats(s.B, s.T, s.planes, s.D), dtype=torch.float32, device=dev)
        s.initial = _ptr(h0); s.states = _ptr(states); s.last = _ptr(last); s.marks = _ptr(marks)
        ws = _workspace(lib, s, 0, dev)
        with L.on_device(dev):
            L.check(lib.gsx_gated_scan_fwd(s, L.stream_ptr(dev)), "gsx_gated_scan_fwd")
        if marks is not None:
            ctx.save_for_backward(gate, x, marks, lengths)
            ctx.how = (form, reverse, initial.dtype if initial is not None else None)
        ctx.set_materialize_grads(False)
        return states, last

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, d_states, d_last):
        gate, x, marks, lengths = ctx.saved_tensors
        form, reverse, initial_dtype = ctx.how
        lib = L.lib()
        dev = x.device
        s = _shape(gate, x, lengths, form, reverse)
        s.marks = _ptr(marks)
        if d_states is not None:
            d_states = _channels(d_states)
            s.d_states = _ptr(d_states)
            s.d_states_stride[:] = [d_states.stride(0), d_states.stride(1), d_states.stride(2) if x.dim() == 4 else 0]
        if d_last is not None:
            d_last = d_last.contiguous()
            s.d_last = _ptr(d_last)
        d_gate = torch.empty(gate.shape, dtype=gate.dtype, device=dev) if ctx.needs_input_grad[0] else None
        d_x = torch.empty(x.shape, dtype=x.dtype, device=dev) if ctx.needs_input_grad[1] else None
        d_initial = torch.empty(x.shape[:1] + x.shape[2:], dtype=torch.float32, device=dev) if ctx.needs_input_grad[2] else None
        s.d_gate = _ptr(d_gate); s.d_x = _ptr(d_x); s.d_initial = _ptr(d_initial)
        ws = _workspace(lib, s, 1, dev)
        with L.on_device(dev):
            L.check(lib.gsx_gated_scan_bwd(s, L.stream_ptr(dev)), "gsx_gated_scan_bwd")
        if d_initial is not None:
            d_initial = d_initial.to(initial_dtype)
        return d_gate, d_x, d_initial, None, None, None, None, None


def _refuse_host(x, name):
    if not x.is_cuda:
        raise RuntimeError(f"gaussian-splatting_amd.{name} runs on an MI355X only (no CPU fallback); use torch ops on CPU tensors")


def _check_pair(gate, x, form):
    if form not in FORMS:
        raise ValueError(f"form must be one of {', '.join(FORMS)}, got {form!r}")
    if x.dtype not in DTYPES or gate.dtype != x.dtype:
        raise TypeError(f"gate and x must share one of float32, bfloat16, float16; got {gate.dtype} and {x.dtype}")
    if gate.device != x.device:
        raise ValueError(f"gate and x must be on one device, got {gate.device} and {x.device}")


def gated_scan(gate, x, initial=None, lengths=None, form="linear", reverse=False, return_states=True):
    """-> (states, last).  x (B, T, D) with gate (B, T, D), or x (B, T, P, D) with gate (B, T, D) shared by P <= 4 planes; one of float32, bfloat16,
    float16.  initial (B, D) / (B, P, D): the state in front of the first step (default zeros); last: the 32-bit state behind the last
    one, to be carried into the next call.  The state is 32 bits all the way; `states` (x's shape and type, None with
    return_states=False) is rounded once.
    lengths (B) int32: sequence b consists of its first lengths[b] steps; what lies behind is not read, states and gradients there are
    zero.  reverse: from step T - 1 (or lengths[b] - 1) down to 0.
    Differentiable once in gate, x and initial; a gate expanded over a batch costs what its full size costs."""
    _check_pair(gate, x, form)
    if gate.dim() != 3 or x.dim() not in (3, 4) or gate.shape != x.shape[:2] + x.shape[-1:]:
        raise ValueError(f"gate (B, T, D) and x (B, T, D) or (B, T, P, D) are wanted, got {tuple(gate.shape)} and {tuple(x.shape)}")
    if x.dim() == 4 and not 1 <= x.shape[2] <= MAX_PLANES:
        raise ValueError(f"1 to {MAX_PLANES} planes can share a gate, got {x.shape[2]}; expand the gate instead")
    if initial is not None and (initial.shape != x.shape[:1] + x.shape[2:] or initial.device != x.device or not initial.is_floating_point()):
        raise ValueError(f"initial must be {tuple(x.shape[:1] + x.shape[2:])} floats on {x.device}, got {tuple(initial.shape)} {initial.dtype} on {initial.device}")
    if lengths is not None:
        if lengths.shape != x.shape[:1] or lengths.device != x.device or lengths.dtype != torch.int32:
            raise ValueError(f"lengths must be ({x.shape[0]},) int32 on {x.device}, got {tuple(lengths.shape)} {lengths.dtype} on {lengths.device}")
        lengths = lengths.contiguous()
    _refuse_host(x, "recurrence")
    want_grad = torch.is_grad_enabled() and (gate.requires_grad or x.requires_grad or (initial is not None and initial.requires_grad))
    return _GatedScan.apply(gate, x, initial, lengths, form, bool(reverse), bool(return_states), want_grad)


@torch.no_grad()
def gated_step(state, gate, x, form="linear"):
    """One step in place on a 32-bit state that lives between calls (a served stream): state, gate, x of one shape, contiguous.  -> state."""
    _check_pair(gate, x, form)
    if state.dtype != torch.float32 or state.shape != x.shape or gate.shape != x.shape or state.device != x.device:
        raise ValueError(f"state (float32), gate and x must share a shape and a device, got {tuple(state.shape)} {state.dtype}, {tuple(gate.shape)}, {tuple(x.shape)}")
    if not state.is_contiguous():
        raise ValueError("gated_step writes the state in place: it must be contiguous")
    _refuse_host(x, "recurrence")
    gate, x = gate.contiguous(), x.contiguous()
    dev = x.device
    with L.on_device(dev):
        L.check(L.lib().gsx_gated_step(DTYPES[x.dtype], FORMS[form], x.numel(), state.data_ptr(), gate.data_ptr(), x.data_ptr(), L.stream_ptr(dev)), "gsx_gated_step")
    torch.autograd.graph.increment_version(state)                # written through a raw pointer: autograd must see it
    return state
