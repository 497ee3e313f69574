"""The gated linear recurrence h_t = a_t h_(t-1) + b_t along one axis as one HIP pass each way (csrc/gsx_gated.hip): the formula by
which depth-ordered splats are composited (/root/reference/model/gaussian_splatting.py:143-144), by itself -- for layers
(render.composite_layers), for decayed traces of per-Gaussian scores over views, for gated sequence models.

    linear   h_t = z_t h_(t-1) + x_t
    blend    h_t = (1 - z_t) h_(t-1) + z_t x_t          (straight colours over each other, z = alpha)
    over     h_t = (1 - z_t) h_(t-1) + x_t              (premultiplied colours)"""
import ctypes as C
import struct
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


def _format(structure):
    """the struct format of a ctypes structure: its fields one after the other, addresses as unsigned words"""
    codes = {C.c_int32: "i", C.c_int64: "q", C.c_void_p: "Q", C.c_size_t: "Q"}
    return "".join(f"{t._length_}{codes[t._type_]}" if hasattr(t, "_length_") else codes[t] for _, t in structure._fields_)


# struct gsx_gated as bytes: filling the ctypes structure field by field takes several times as long
_PACK = struct.Struct(_format(L.GsxGated)).pack
_entry = None


def _entries():
    """(workspace, forward, backward) that take the packed struct; the table is whole before another thread can see it"""
    global _entry
    if _entry is None:
        lib, entry = L.lib(), {}
        for name, argtypes, restype in (("gsx_gated_workspace_bytes", [C.c_char_p, C.c_int32], C.c_size_t),
                                        ("gsx_gated_scan_fwd", [C.c_char_p, C.c_void_p], C.c_int), ("gsx_gated_scan_bwd", [C.c_char_p, C.c_void_p], C.c_int)):
            fn = lib[name]                                       # a function object of its own: the binding's keeps its types
            fn.argtypes, fn.restype = argtypes, restype
            entry[name] = fn
        _entry = entry
    return _entry


def _call(name, backward, head, tail, dev):
    e = _entries()
    packed = _PACK(*head, *tail, 0, 0)
    n = e["gsx_gated_workspace_bytes"](packed, backward)
    if n:
        ws = torch.empty(n, dtype=torch.uint8, device=dev)
        packed = _PACK(*head, *tail, ws.data_ptr(), n)
    with L.on_device(dev):
        L.check(e[name](packed, L.stream_ptr(dev)), name)


def _head(gate, x, initial, lengths, form, reverse):
    gs, xs = gate.stride(), x.stride()
    B, T, D = gate.shape
    four = x.dim() == 4
    return (DTYPES[x.dtype], FORMS[form], reverse, x.shape[2] if four else 1, B, T, D, gate.data_ptr(), gs[0], gs[1],
            x.data_ptr(), xs[0], xs[1], xs[2] if four else 0, initial.data_ptr() if initial is not None else 0, lengths.data_ptr() if lengths is not None else 0)


class _GatedScan(torch.autograd.Function):
    @staticmethod
    def forward(ctx, gate, x, initial, lengths, form, reverse, want_states, want_grad):
        gate, x = _channels(gate), _channels(x)
        dev = x.device
        state_shape = x.shape[:1] + x.shape[2:]
        h0 = initial.to(torch.float32).contiguous() if initial is not None else None
        states = torch.empty(x.shape, dtype=x.dtype, device=dev) if want_states else None
        last = torch.empty(state_shape, dtype=torch.float32, device=dev)
        head = _head(gate, x, h0, lengths, form, reverse)
        marks = None
        if want_grad:
            n = L.lib().gsx_gated_marks_floats(head[4], head[5], head[3], head[6])
            if n < 0:
                L.check(n, "gsx_gated_marks_floats")
            marks = torch.empty(n, dtype=torch.float32, device=dev)
        _call("gsx_gated_scan_fwd", 0, head, (states.data_ptr() if want_states else 0, last.data_ptr(), marks.data_ptr() if want_grad else 0,
                                              0, 0, 0, 0, 0, 0, 0, 0), dev)
        if want_grad:
            ctx.save_for_backward(gate, x, marks, lengths)
            ctx.how = (form, reverse, initial.dtype if initial is not None else None)
        ctx.set_materialize_grads(False)
        return states, last

    @staticmethod
    def backward(ctx, d_states, d_last):
        if torch.is_grad_enabled():                              # create_graph: the gradients' own gradients are not here
            raise RuntimeError("gated_scan is differentiable once only")
        gate, x, marks, lengths = ctx.saved_tensors
        form, reverse, initial_dtype = ctx.how
        need = ctx.needs_input_grad
        dev = x.device
        ds = (0, 0, 0)
        if d_states is not None:
            d_states = _channels(d_states)
            st = d_states.stride()
            ds = (st[0], st[1], st[2] if x.dim() == 4 else 0)
        if d_last is not None:
            d_last = d_last.contiguous()
        d_gate = torch.empty(gate.shape, dtype=gate.dtype, device=dev) if need[0] else None
        d_x = torch.empty(x.shape, dtype=x.dtype, device=dev) if need[1] else None
        d_initial = torch.empty(x.shape[:1] + x.shape[2:], dtype=torch.float32, device=dev) if need[2] else None
        at = lambda t: t.data_ptr() if t is not None else 0  # noqa: E731
        _call("gsx_gated_scan_bwd", 1, _head(gate, x, None, lengths, form, reverse),
              (0, 0, marks.data_ptr(), at(d_states), *ds, at(d_last), at(d_gate), at(d_x), at(d_initial)), dev)
        if d_initial is not None and initial_dtype != torch.float32:
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
    Differentiable once in gate, x and initial; a gate expanded over a batch costs what its full size costs.  Can be captured into a graph; capture
    its backward with torch.autograd.grad, or while no earlier graph of the same leaves is alive (torch would accumulate on that one's stream)."""
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


def gated_step(state, gate, x, form="linear"):
    """One step in place on a 32-bit state that lives between calls (a served stream): state, gate, x of one shape, contiguous; gate and x may be
    the state itself, but may not overlap it otherwise.  -> state.
    Not differentiable (gated_scan with one step is): under grad mode, arguments that require a gradient are refused."""
    _check_pair(gate, x, form)
    shape = state.shape
    if state.dtype != torch.float32 or shape != x.shape or gate.shape != shape or state.device != x.device:
        raise ValueError(f"state (float32), gate and x must share a shape and a device, got {tuple(state.shape)} {state.dtype}, {tuple(gate.shape)}, {tuple(x.shape)}")
    if not state.is_contiguous():
        raise ValueError("gated_step writes the state in place: it must be contiguous")
    if (state.requires_grad or gate.requires_grad or x.requires_grad) and torch.is_grad_enabled():
        raise RuntimeError("gated_step writes the state in place and leaves no graph: state, gate and x must not require a gradient")
    _refuse_host(x, "recurrence")
    gate, x = gate.contiguous(), x.contiguous()
    dev = x.device
    with L.on_device(dev):
        L.check(L.lib().gsx_gated_step(DTYPES[x.dtype], FORMS[form], x.numel(), state.data_ptr(), gate.data_ptr(), x.data_ptr(), L.stream_ptr(dev)), "gsx_gated_step")
    torch._C._increment_version((state,))                        # written through a raw pointer: autograd must see it
    return state
