"""Draws from softmax(logits / temperature) by given random numbers (csrc/gsx_draw.hip): what GaussianSplat.get_dense_points does with a
scene's opacities (/root/reference/model/gaussian_splatting.py:420-443), with the cuts by rank, mass and share, for one row of
millions of Gaussians as for many rows (a layer per pixel, a batch of a large alphabet)."""
import math
import torch
from . import _lib as L
from .recurrence import DTYPES, _ptr, _refuse_host

LEAST = 2.0 ** -126                                              # the smallest normal number of 32 bits
WIDE = (torch.int64, torch.uint32, torch.uint64)
MAX_V = 1 << 27                                                  # GSX_DRAW_MAX_V


def _setting(v, name, R, device, dtype, ok, where, positive=False):
    """(number, tensor): a setting of all rows, or one per row; positive: one above 0 stays above 0 in 32 bits"""
    if torch.is_tensor(v):
        if v.shape != (R,) or v.device != device:
            raise ValueError(f"{name} must be a number or ({R},) on {device}, got {tuple(v.shape)} on {v.device}")
        if dtype == torch.int32 and (v.is_floating_point() or v.is_complex()):
            raise TypeError(f"{name} by row must be whole numbers, got {v.dtype}")
        v = v.detach()
        if dtype == torch.int32 and v.dtype in WIDE:
            v = v.to(torch.int64).clamp(-1, MAX_V)               # all tokens and more, where a cast alone would wrap (from 2^63 on it is negative: all)
        if positive and v.dtype == torch.float64:
            v = torch.where(v > 0, v.clamp(min=LEAST), v)
        return 0, v.to(dtype).contiguous()
    if not ok(v):
        raise ValueError(f"{name} must be {where}, got {v}")
    return (max(v, LEAST) if positive and v > 0 else v), None


@torch.no_grad()
def sample(logits, uniforms, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, return_logprobs=False):
    """logits (R, V) float32 / bfloat16 / float16, uniforms (R, S) float32 or float64 in [0, 1) -> indices (R, S) int64 (and their log
    probabilities, float32).  Tokens are ranked by (logit descending, index ascending); kept are the first top_k (0: all), of these the
    fewest whose mass reaches top_p of their mass, of these the ones at least min_p times as likely as the first.  A draw is the lowest
    index whose inclusive kept mass, in index order, exceeds u times all kept mass (u of 1 and more: the largest double below 1; below 0 and NaN: 0).
    temperature (0: the lowest index of the largest logit), top_k, top_p and min_p are numbers or tensors of one value per row, taken in 32 bits (what is above 0 stays so).  NaN and -inf logits
    are masked; a row with nothing left, or with a value of its own out of range, gives -1 (and -inf).  float32 uniforms have 24 bits:
    take float64 where V is in the millions.  V is 2^27 at most, 524284 for more than 65535 rows.  Not differentiable."""
    if logits.dim() != 2 or uniforms.dim() != 2 or uniforms.shape[0] != logits.shape[0]:
        raise ValueError(f"logits (R, V) and uniforms (R, S) are wanted, got {tuple(logits.shape)} and {tuple(uniforms.shape)}")
    if logits.dtype not in DTYPES or uniforms.dtype not in (torch.float32, torch.float64):
        raise TypeError(f"logits must be float32, bfloat16 or float16 and uniforms float32 or float64, got {logits.dtype} and {uniforms.dtype}")
    if uniforms.device != logits.device:
        raise ValueError(f"logits and uniforms must be on one device, got {logits.device} and {uniforms.device}")
    R, V = logits.shape
    S = uniforms.shape[1]
    if V > MAX_V:
        raise ValueError(f"a row may have {MAX_V} tokens, got {V}")
    dev = logits.device
    t, ts = _setting(temperature, "temperature", R, dev, torch.float32, lambda v: v >= 0, "0 or more", positive=True)
    k, ks = _setting(top_k, "top_k", R, dev, torch.int32, lambda v: 0 <= v < math.inf and v == int(v), "a whole number, 0 or more")
    p, ps = _setting(top_p, "top_p", R, dev, torch.float32, lambda v: v > 0, "above 0", positive=True)
    m, ms = _setting(min_p, "min_p", R, dev, torch.float32, lambda v: 0 <= v <= 1, "in [0, 1]")
    _refuse_host(logits, "sampling")
    lib = L.lib()
    logits = logits.detach()
    logits = logits if V <= 1 or logits.stride(1) == 1 else logits.contiguous()
    uniforms = uniforms.contiguous()
    indices = torch.empty((R, S), dtype=torch.int64, device=dev)
    logprobs = torch.empty((R, S), dtype=torch.float32, device=dev) if return_logprobs else None
    s = L.GsxDraw()
    s.dtype = DTYPES[logits.dtype]; s.uniforms_f64 = int(uniforms.dtype == torch.float64)
    s.R, s.V, s.S = R, V, S
    s.logits = _ptr(logits); s.row_stride = logits.stride(0); s.uniforms = _ptr(uniforms)
    s.temperature, s.top_k, s.top_p, s.min_p = t, min(int(k), V), p, m
    s.temperatures, s.top_ks, s.top_ps, s.min_ps = _ptr(ts), _ptr(ks), _ptr(ps), _ptr(ms)
    s.indices = _ptr(indices); s.logprobs = _ptr(logprobs)
    if R and S:
        ws = torch.empty(lib.gsx_draw_workspace_bytes(s), dtype=torch.uint8, device=dev)
        s.ws = _ptr(ws); s.ws_bytes = ws.numel()
        with L.on_device(dev):
            L.check(lib.gsx_draw_indices(s, L.stream_ptr(dev)), "gsx_draw_indices")
    return (indices, logprobs) if return_logprobs else indices
