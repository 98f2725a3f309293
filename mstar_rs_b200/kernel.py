"""Torch-tensor front end of the sampler kernel.

`sampler_step` fills a `Params` struct from device tensors and launches one
sampling step on the current CUDA stream.  It allocates nothing, never
synchronises and never reads device memory on the host, so it can be called
inside `torch.cuda.graph` capture.  Shapes, dtypes, devices and contiguity are
validated here (before any launch) and again by the C ABI.
"""
from __future__ import annotations

import ctypes
import functools

import torch

from . import _native as N

_DT = {torch.float32: N.DTYPE_F32, torch.bfloat16: N.DTYPE_BF16}
_U64 = (torch.int64, torch.uint64)  # seed / offset: 64-bit words, read as unsigned


def _ptr(t):
    return None if t is None else ctypes.c_void_p(t.data_ptr())


def _need(t, name, dtype, dev, shape0=None, ndim=1):
    if t is None:
        return
    ok = dtype if isinstance(dtype, tuple) else (dtype,)
    if t.dtype not in ok:
        raise TypeError(f"{name} must be {dtype}, got {t.dtype}")
    if t.device != dev:
        raise ValueError(f"{name} must live on {dev}, got {t.device}")
    if t.dim() != ndim:
        raise ValueError(f"{name} must be {ndim}-D, got shape {tuple(t.shape)}")
    if not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous")
    if shape0 is not None and t.shape[0] < shape0:
        raise ValueError(f"{name} has {t.shape[0]} rows, need >= {shape0}")


def build_params(logits: torch.Tensor, *, slot_idx=None, num_slots=None, temperature=None, top_k=None,
                 top_p=None, min_p=None, rep_pen=None, pres_pen=None, freq_pen=None, hist_ids=None,
                 hist_len=None, seen_bits=None, seen_cap=0, bias_ids=None, bias_vals=None,
                 allowed_bits=None, uniforms=None, seed=None, offset=None, out_ids=None, out_ids32=None,
                 out_status=None, out_x=None, out_kept=None, out_probs=None, flags=0, cluster_size=0,
                 vocab_offset=0, stop_ids=None, stop_flags=None) -> N.Params:
    if logits.dim() != 2:
        raise ValueError("logits must be [B, V]")
    if logits.dtype not in _DT:
        raise TypeError(f"logits must be float32 or bfloat16, got {logits.dtype}")
    if not logits.is_cuda:
        raise ValueError("logits must be a CUDA tensor (there is no CPU path)")
    if logits.stride(1) != 1:
        raise ValueError("logits rows must be contiguous")
    dev = logits.device
    B, V = logits.shape
    ns = num_slots
    if ns is None:
        for t in (temperature, top_k, top_p, min_p, rep_pen, pres_pen, freq_pen, seed, offset, hist_len):
            if t is not None:
                ns = t.shape[0]
                break
        else:
            ns = B
    _need(slot_idx, "slot_idx", torch.int32, dev, B)
    for name, t, dt in (("temperature", temperature, torch.float32), ("top_k", top_k, torch.int32),
                        ("top_p", top_p, torch.float32), ("min_p", min_p, torch.float32),
                        ("rep_pen", rep_pen, torch.float32), ("pres_pen", pres_pen, torch.float32),
                        ("freq_pen", freq_pen, torch.float32), ("hist_len", hist_len, torch.int32),
                        ("seed", seed, _U64), ("offset", offset, _U64)):
        _need(t, name, dt, dev, ns)
    _need(hist_ids, "hist_ids", torch.int32, dev, ns, 2)
    _need(seen_bits, "seen_bits", torch.int32, dev, ns, 2)
    _need(bias_ids, "bias_ids", torch.int32, dev, ns, 2)
    _need(bias_vals, "bias_vals", torch.float32, dev, ns, 2)
    _need(allowed_bits, "allowed_bits", torch.int32, dev, ns, 2)
    _need(stop_ids, "stop_ids", torch.int32, dev, ns, 2)
    _need(stop_flags, "stop_flags", torch.int32, dev, ns)
    if stop_flags is not None and stop_ids is None:
        raise ValueError("stop_flags needs stop_ids")
    _need(uniforms, "uniforms", torch.float32, dev, B)
    _need(out_ids, "out_ids", torch.int64, dev, B)
    _need(out_ids32, "out_ids32", torch.int32, dev, B)
    _need(out_status, "out_status", torch.int32, dev, B)
    for name, t, dt in (("out_x", out_x, torch.float32), ("out_kept", out_kept, torch.uint8),
                        ("out_probs", out_probs, torch.float32)):
        if t is not None:
            _need(t, name, dt, dev, B, 2)
            if t.shape[1] != V:
                raise ValueError(f"{name} must be [B, V]")
    p = N.Params()
    p.logits = logits.data_ptr()
    p.dtype = _DT[logits.dtype]
    p.B, p.V, p.num_slots = B, V, ns
    p.ld = logits.stride(0)
    p.vocab_offset = vocab_offset
    p.slot_idx = _ptr(slot_idx)
    p.temperature, p.top_k, p.top_p, p.min_p = _ptr(temperature), _ptr(top_k), _ptr(top_p), _ptr(min_p)
    p.rep_pen, p.pres_pen, p.freq_pen = _ptr(rep_pen), _ptr(pres_pen), _ptr(freq_pen)
    p.hist_ids, p.hist_len = _ptr(hist_ids), _ptr(hist_len)
    p.H = 0 if hist_ids is None else hist_ids.shape[1]
    p.seen_cap = seen_cap
    p.seen_bits = _ptr(seen_bits)
    p.seen_words = 0 if seen_bits is None else seen_bits.shape[1]
    p.bias_ids, p.bias_vals = _ptr(bias_ids), _ptr(bias_vals)
    p.NB = 0 if bias_ids is None else bias_ids.shape[1]
    p.allowed_bits = _ptr(allowed_bits)
    p.allowed_words = 0 if allowed_bits is None else allowed_bits.shape[1]
    p.uniforms, p.seed, p.offset = _ptr(uniforms), _ptr(seed), _ptr(offset)
    p.out_ids, p.out_ids32, p.out_status = _ptr(out_ids), _ptr(out_ids32), _ptr(out_status)
    p.out_x, p.out_kept, p.out_probs = _ptr(out_x), _ptr(out_kept), _ptr(out_probs)
    p.flags = flags
    p.cluster_size = cluster_size
    p.stop_ids = _ptr(stop_ids)
    p.NS = 0 if stop_ids is None else stop_ids.shape[1]
    p.stop_flags = _ptr(stop_flags)
    return p


def launch_step(p: N.Params, device: torch.device) -> None:
    with torch.cuda.device(device):
        stream = torch.cuda.current_stream(device).cuda_stream
        N.check(N.lib().mstar_sampler_step(ctypes.byref(p), ctypes.c_void_p(stream)), "mstar_sampler_step")


def sampler_step(logits: torch.Tensor, **kw) -> N.Params:
    """Launch one sampling step; returns the Params used (keep it to relaunch)."""
    p = build_params(logits, **kw)
    launch_step(p, logits.device)
    return p


def sampler_step_heads(logits: torch.Tensor, **kw) -> N.Params:
    """One launch for H heads of n rows each (logits [H, n, V], e.g. the
    codebook heads of a multi-codebook decoder sampled together): row h * n + i
    of the flattened [H * n, V] batch is head h's row i, and slot_idx [H * n]
    (or the row number) picks its parameters and per-slot state, so each
    (head, request) pair keeps its own history, seen mask and RNG offset."""
    if logits.dim() != 3:
        raise ValueError("logits must be [H, n, V]")
    H, n, V = logits.shape
    if logits.stride(2) != 1 or logits.stride(0) != n * logits.stride(1):
        raise ValueError("logits heads must be stacked rows of one [H * n, V] matrix")
    return sampler_step(logits.reshape(H * n, V), **kw)


def plan(logits: torch.Tensor, **kw):
    p = build_params(logits, **kw)
    cs, sm = N.I32(), N.I64()
    N.check(N.lib().mstar_sampler_plan(ctypes.byref(p), ctypes.byref(cs), ctypes.byref(sm)), "mstar_sampler_plan")
    return cs.value, sm.value


def tp_record_words(tp_cap: int) -> int:
    return int(N.lib().mstar_sampler_tp_record_words(tp_cap))


def tp_local(logits: torch.Tensor, tp_cap: int, send: torch.Tensor, **kw) -> None:
    p = build_params(logits, **kw)
    if send.dtype != torch.int32 or not send.is_contiguous() or send.device != logits.device:
        raise ValueError("send must be a contiguous int32 tensor on the logits device")
    if send.numel() < logits.shape[0] * tp_record_words(tp_cap):
        raise ValueError("send buffer too small")
    with torch.cuda.device(logits.device):
        stream = torch.cuda.current_stream(logits.device).cuda_stream
        N.check(N.lib().mstar_sampler_tp_local(ctypes.byref(p), tp_cap, ctypes.c_void_p(send.data_ptr()),
                                               ctypes.c_void_p(stream)), "mstar_sampler_tp_local")


def tp_merge(logits: torch.Tensor, tp_cap: int, tp_world: int, V_global: int, recv: torch.Tensor, **kw) -> None:
    p = build_params(logits, **kw)
    if recv.dtype != torch.int32 or not recv.is_contiguous() or recv.device != logits.device:
        raise ValueError("recv must be a contiguous int32 tensor on the logits device")
    if recv.numel() < tp_world * logits.shape[0] * tp_record_words(tp_cap):
        raise ValueError("recv buffer too small")
    with torch.cuda.device(logits.device):
        stream = torch.cuda.current_stream(logits.device).cuda_stream
        N.check(N.lib().mstar_sampler_tp_merge(ctypes.byref(p), tp_cap, tp_world, V_global,
                                               ctypes.c_void_p(recv.data_ptr()), ctypes.c_void_p(stream)),
                "mstar_sampler_tp_merge")


def _u32(t, name, dev, n):
    if t.dtype != torch.int32 or t.device != dev or not t.is_contiguous() or t.numel() < n:
        raise ValueError(f"{name} must be a contiguous int32 tensor of >= {n} words on {dev}")


def tp_local2(logits: torch.Tensor, tp_cap: int, send: torch.Tensor, xbuf: torch.Tensor, **kw) -> None:
    """Two-round shard records (mstar_sampler_tp_local2): rows without a
    usable top_k send their first tp_cap members and leave their shard
    values in xbuf [B, V] float32."""
    p = build_params(logits, **kw)
    dev = logits.device
    _u32(send, "send", dev, logits.shape[0] * tp_record_words(tp_cap))
    if xbuf.dtype != torch.float32 or xbuf.device != dev or not xbuf.is_contiguous() or \
            xbuf.numel() < logits.shape[0] * logits.shape[1]:
        raise ValueError("xbuf must be a contiguous float32 [B, V] tensor on the logits device")
    with torch.cuda.device(dev):
        stream = torch.cuda.current_stream(dev).cuda_stream
        N.check(N.lib().mstar_sampler_tp_local2(ctypes.byref(p), tp_cap, _ptr(send), _ptr(xbuf),
                                                ctypes.c_void_p(stream)), "mstar_sampler_tp_local2")


def tp_merge1(logits: torch.Tensor, tp_cap: int, tp_world: int, V_global: int, recv: torch.Tensor,
              pend: torch.Tensor, **kw) -> None:
    """First merge of the two-round exchange (mstar_sampler_tp_merge1): decides
    the rows no shard cut short, defers the others into pend [B, 2] int32."""
    p = build_params(logits, **kw)
    dev = logits.device
    B = logits.shape[0]
    _u32(recv, "recv", dev, tp_world * B * tp_record_words(tp_cap))
    _u32(pend, "pend", dev, 2 * B)
    with torch.cuda.device(dev):
        stream = torch.cuda.current_stream(dev).cuda_stream
        N.check(N.lib().mstar_sampler_tp_merge1(ctypes.byref(p), tp_cap, tp_world, V_global, _ptr(recv), _ptr(pend),
                                                ctypes.c_void_p(stream)), "mstar_sampler_tp_merge1")


def tp_mass(logits: torch.Tensor, xbuf: torch.Tensor, pend: torch.Tensor, send2: torch.Tensor, **kw) -> None:
    """The shard's exact A mass of every deferred row (mstar_sampler_tp_mass)
    into send2 [B, 2] int32 (a little-endian u64 per row)."""
    p = build_params(logits, **kw)
    dev = logits.device
    B = logits.shape[0]
    _u32(pend, "pend", dev, 2 * B)
    _u32(send2, "send2", dev, 2 * B)
    with torch.cuda.device(dev):
        stream = torch.cuda.current_stream(dev).cuda_stream
        N.check(N.lib().mstar_sampler_tp_mass(ctypes.byref(p), _ptr(xbuf), _ptr(pend), _ptr(send2),
                                              ctypes.c_void_p(stream)), "mstar_sampler_tp_mass")


def tp_merge2(logits: torch.Tensor, tp_cap: int, tp_world: int, V_global: int, recv: torch.Tensor,
              recv2: torch.Tensor, pend: torch.Tensor, **kw) -> None:
    """Second merge of the two-round exchange (mstar_sampler_tp_merge2)."""
    p = build_params(logits, **kw)
    dev = logits.device
    B = logits.shape[0]
    _u32(recv, "recv", dev, tp_world * B * tp_record_words(tp_cap))
    _u32(recv2, "recv2", dev, tp_world * 2 * B)
    _u32(pend, "pend", dev, 2 * B)
    with torch.cuda.device(dev):
        stream = torch.cuda.current_stream(dev).cuda_stream
        N.check(N.lib().mstar_sampler_tp_merge2(ctypes.byref(p), tp_cap, tp_world, V_global, _ptr(recv), _ptr(recv2),
                                                _ptr(pend), ctypes.c_void_p(stream)), "mstar_sampler_tp_merge2")


def commit(ids: torch.Tensor, *, V: int, num_slots: int, slot_idx=None, hist_ids=None, hist_len=None,
           seen_bits=None, stop_ids=None, stop_flags=None, offset=None, flags=0, vocab_offset=0) -> None:
    """Per-slot state updates for ids chosen elsewhere (mstar_sampler_commit):
    history append / seen bit / RNG offset as `flags` selects, stop flags."""
    if ids.dtype != torch.int64 or ids.dim() != 1 or not ids.is_cuda or not ids.is_contiguous():
        raise ValueError("ids must be a contiguous 1-D int64 CUDA tensor")
    dev = ids.device
    B = ids.shape[0]
    _need(slot_idx, "slot_idx", torch.int32, dev, B)
    _need(hist_len, "hist_len", torch.int32, dev, num_slots)
    _need(offset, "offset", _U64, dev, num_slots)
    _need(stop_flags, "stop_flags", torch.int32, dev, num_slots)
    _need(hist_ids, "hist_ids", torch.int32, dev, num_slots, 2)
    _need(seen_bits, "seen_bits", torch.int32, dev, num_slots, 2)
    _need(stop_ids, "stop_ids", torch.int32, dev, num_slots, 2)
    p = N.Params()
    p.B, p.V, p.num_slots, p.vocab_offset = B, V, num_slots, vocab_offset
    p.slot_idx = _ptr(slot_idx)
    p.hist_ids, p.hist_len = _ptr(hist_ids), _ptr(hist_len)
    p.H = 0 if hist_ids is None else hist_ids.shape[1]
    p.seen_bits = _ptr(seen_bits)
    p.seen_words = 0 if seen_bits is None else seen_bits.shape[1]
    p.stop_ids, p.stop_flags = _ptr(stop_ids), _ptr(stop_flags)
    p.NS = 0 if stop_ids is None else stop_ids.shape[1]
    p.offset = _ptr(offset)
    p.flags = flags
    with torch.cuda.device(dev):
        stream = torch.cuda.current_stream(dev).cuda_stream
        N.check(N.lib().mstar_sampler_commit(ctypes.byref(p), ctypes.c_void_p(ids.data_ptr()),
                                             ctypes.c_void_p(stream)), "mstar_sampler_commit")


def _check_lmhead(hidden: torch.Tensor, weight: torch.Tensor):
    if hidden.dtype != torch.bfloat16 or weight.dtype != torch.bfloat16:
        raise TypeError("hidden and weight must be bfloat16")
    if not hidden.is_cuda or weight.device != hidden.device:
        raise ValueError("hidden and weight must be CUDA tensors on one device")
    if hidden.dim() != 2 or weight.dim() != 2 or hidden.shape[1] != weight.shape[1]:
        raise ValueError("hidden must be [B, d] and weight [V, d]")
    if not hidden.is_contiguous() or not weight.is_contiguous():
        raise ValueError("hidden and weight must be contiguous")
    return hidden.shape[0], weight.shape[0], hidden.shape[1]


_WS: dict = {}


def lmhead_workspace(B: int, device: torch.device) -> torch.Tensor:
    """Scratch for projections of up to B rows on `device`
    (mstar_lmhead_workspace_bytes), kept per device and reused: calls on one
    stream share it; give each concurrent stream its own."""
    dev = torch.device(device)
    with torch.cuda.device(dev):
        n = int(N.lib().mstar_lmhead_workspace_bytes(B))
    if n <= 0:
        raise ValueError(f"B={B} is outside [1, 256]")
    key = dev.index if dev.index is not None else torch.cuda.current_device()
    ws = _WS.get(key)
    if ws is None or ws.numel() < n:
        ws = torch.empty(n, dtype=torch.uint8, device=dev)
        _WS[key] = ws
    return ws


def _check_ws(ws, dev):
    if ws is None:
        return None, 0
    if ws.dtype != torch.uint8 or ws.device != dev or not ws.is_contiguous():
        raise ValueError("workspace must be a contiguous uint8 tensor on the hidden device")
    return _ptr(ws), ws.numel()


def lmhead_logits(hidden: torch.Tensor, weight: torch.Tensor, *, out: torch.Tensor | None = None,
                  dtype=torch.float32, status: torch.Tensor | None = None, workspace="auto") -> torch.Tensor:
    """hidden [B, d] @ weight[V, d]^T on the tensor cores (mstar_lmhead_logits),
    fp32 accumulation, stored as float32 or bfloat16.  workspace: "auto" (the
    device's cached lmhead_workspace), a uint8 tensor, or None (whole-tile
    shares, no scratch)."""
    B, V, d = _check_lmhead(hidden, weight)
    dev = hidden.device
    if out is None:
        out = torch.empty(B, V, dtype=dtype, device=dev)
    if out.dtype not in _DT or out.device != dev or out.dim() != 2 or out.shape[0] != B or out.shape[1] < V \
            or out.stride(1) != 1:
        raise ValueError("out must be [B, >= V] float32 / bfloat16 with contiguous rows on the hidden device")
    if status is not None and (status.dtype != torch.int32 or status.device != dev or status.numel() < 1):
        raise ValueError("status must be an int32 tensor on the hidden device")
    if isinstance(workspace, str):
        workspace = lmhead_workspace(B, dev)
    wp, wn = _check_ws(workspace, dev)
    with torch.cuda.device(dev):
        stream = torch.cuda.current_stream(dev).cuda_stream
        N.check(N.lib().mstar_lmhead_logits(_ptr(hidden), _ptr(weight), B, V, d, _ptr(out), _DT[out.dtype],
                                            out.stride(0), wp, wn, _ptr(status), ctypes.c_void_p(stream)),
                "mstar_lmhead_logits")
    return out


def lmhead_step(hidden: torch.Tensor, weight: torch.Tensor, logits: torch.Tensor, *, status=None,
                workspace="auto", **kw) -> N.Params:
    """Project hidden [B, d] by weight [V, d] into `logits` [B, V] (float32 or
    bfloat16, written) and sample from it (mstar_sampler_lmhead_step).  The
    sampling keywords are sampler_step's; workspace as for lmhead_logits."""
    B, V, d = _check_lmhead(hidden, weight)
    if logits.shape[0] != B or logits.dim() != 2 or logits.shape[1] != V:
        raise ValueError("logits must be [B, V] for hidden [B, d] and weight [V, d]")
    if status is not None and (status.dtype != torch.int32 or status.device != hidden.device or status.numel() < 1):
        raise ValueError("status must be an int32 tensor on the hidden device")
    p = build_params(logits, **kw)
    if isinstance(workspace, str):
        workspace = lmhead_workspace(B, hidden.device)
    wp, wn = _check_ws(workspace, hidden.device)
    with torch.cuda.device(logits.device):
        stream = torch.cuda.current_stream(logits.device).cuda_stream
        N.check(N.lib().mstar_sampler_lmhead_step(ctypes.byref(p), _ptr(hidden), _ptr(weight), d, wp, wn,
                                                  _ptr(status), ctypes.c_void_p(stream)),
                "mstar_sampler_lmhead_step")
    return p


# ------------------------------------------------- 4-bit weights, lookup, log-probabilities, policy loss

_FN: dict = {}  # entry points by name, once the library is loaded


def _call(dev: torch.device, name: str, *args) -> None:
    """Entry point `name` with `args` and the current stream of `dev`, on `dev`."""
    fn = _FN.get(name)
    if fn is None:
        fn = _FN[name] = getattr(N.lib(), name)
    if torch.cuda.current_device() == dev.index:
        rc = fn(*args, _raw_stream(dev.index))
    else:
        with torch.cuda.device(dev):
            rc = fn(*args, _raw_stream(dev.index))
    if rc != N.OK:
        N.check(rc, name)


def _raw_stream(index: int) -> int:
    return torch.cuda.current_stream(index).cuda_stream


if hasattr(torch._C, "_cuda_getCurrentRawStream"):  # the same handle without the Stream object around it
    _raw_stream = torch._C._cuda_getCurrentRawStream  # noqa: F811


def _cuda(t: torch.Tensor, name: str) -> torch.device:
    if not t.is_cuda:
        raise ValueError(f"{name} must be a CUDA tensor (there is no CPU path)")
    return t.device


def _vec(t, name, dtype, dev, n):
    """The address of a contiguous [n] tensor of `dtype` (None: NULL)."""
    if t is None:
        return None
    if t.dtype is dtype and t.dim() == 1 and t.shape[0] == n and t.is_contiguous() and t.device == dev:
        return t.data_ptr()
    if t.dtype != dtype:
        raise TypeError(f"{name} must be {dtype}, got {t.dtype}")
    if t.device != dev:
        raise ValueError(f"{name} must live on {dev}, got {t.device}")
    raise ValueError(f"{name} must be a contiguous [{n}] tensor, got shape {tuple(t.shape)}")


def _status(t, dev):
    if t is None:
        return None
    if t.dtype != torch.int32 or t.device != dev or t.numel() < 1:
        raise ValueError(f"status must be an int32 tensor on {dev}")
    return t.data_ptr()


def _matrix(t, name, dev, rows, cols):
    """Checks a [rows, cols] float32 / bfloat16 matrix with contiguous rows."""
    if t.dtype in _DT and t.dim() == 2 and t.shape[0] == rows and t.shape[1] == cols and t.is_contiguous() \
            and t.device == dev:
        return
    if t.dtype not in _DT:
        raise TypeError(f"{name} must be float32 or bfloat16, got {t.dtype}")
    if t.device != dev:
        raise ValueError(f"{name} must live on {dev}, got {t.device}")
    if t.dim() != 2 or t.shape[0] != rows or t.shape[1] != cols or (t.stride(1) != 1 and cols > 1):
        raise ValueError(f"{name} must be [{rows}, {cols}] with contiguous rows, got shape {tuple(t.shape)} "
                         f"with strides {t.stride()}")
    if rows > 1 and t.stride(0) < cols:
        raise ValueError(f"{name}'s rows overlap (row stride {t.stride(0)})")


def _ld(t) -> int:
    return t.stride(0) if t.shape[0] > 1 else max(t.stride(0), t.shape[1])


def _span(t: torch.Tensor) -> int:
    """Bytes from a tensor's first element to behind its last."""
    if t.numel() == 0:
        return 0
    return (sum((n - 1) * s for n, s in zip(t.shape, t.stride())) + 1) * t.element_size()


def _overlap(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Whether two matrices' memory ranges meet without being the same rows."""
    if a.data_ptr() == b.data_ptr() and _ld(a) == _ld(b) and a.dtype == b.dtype:
        return False
    a0, b0 = a.data_ptr(), b.data_ptr()
    return a0 < b0 + _span(b) and b0 < a0 + _span(a)


def quantize_w4(weight: torch.Tensor, group_size: int = 128, *, zero_points: bool = False, scale_dtype=torch.bfloat16):
    """Round a [V, d] weight to 4 bits with one scale per row and group of
    `group_size` columns: (codes [V, d / 2] uint8, the even column in the low
    four bits; scales [V, d / group_size]; zeros uint8 or None).  Without zero
    points codes run from -8 to 7 about 8; with them each group's range maps
    to 0 .. 15.  A one-time step on any device (plain tensor operations)."""
    if weight.dim() != 2:
        raise ValueError("weight must be [V, d]")
    if group_size not in (32, 64, 128) or weight.shape[1] % group_size:
        raise ValueError("group_size must be 32, 64 or 128 and divide d")
    if scale_dtype not in _DT:
        raise TypeError("scale_dtype must be float32 or bfloat16")
    V, d = weight.shape
    w = weight.detach().float().contiguous().view(V, d // group_size, group_size)
    if zero_points:
        lo, hi = w.amin(2).clamp(max=0), w.amax(2).clamp(min=0)
        scales = ((hi - lo) / 15).to(scale_dtype)
    else:
        scales = (w.abs().amax(2) / 7.5).to(scale_dtype)
    s = scales.float()
    s = torch.where(s > 0, s, 1.0)
    zeros = (-lo / s).round().clamp(0, 15) if zero_points else torch.full_like(s, 8.0)
    q = (w / s[:, :, None] + zeros[:, :, None]).round().clamp(0, 15).to(torch.uint8).view(V, d)
    return q[:, 0::2] | (q[:, 1::2] << 4), scales, zeros.to(torch.uint8) if zero_points else None


def _w4(codes, scales, zeros) -> N.W4:
    dev = _cuda(codes, "codes")
    if codes.dtype != torch.uint8 or codes.dim() != 2 or not codes.is_contiguous():
        raise ValueError("codes must be a contiguous [V, d / 2] uint8 tensor")
    if scales.dtype not in _DT:
        raise TypeError(f"scales must be float32 or bfloat16, got {scales.dtype}")
    V, d = codes.shape[0], codes.shape[1] * 2
    if scales.device != dev or scales.dim() != 2 or scales.shape[0] != V or not scales.is_contiguous():
        raise ValueError("scales must be a contiguous [V, d / group] tensor on the codes' device")
    G = scales.shape[1]
    if G < 1 or d % G or d // G not in (32, 64, 128):
        raise ValueError(f"scales give groups of {d / max(G, 1):g} columns; they must be of 32, 64 or 128")
    zp = None
    if zeros is not None:
        if zeros.dtype != torch.uint8 or zeros.device != dev or zeros.shape != scales.shape or not zeros.is_contiguous():
            raise ValueError("zeros must be a contiguous uint8 tensor of the scales' shape on their device")
        zp = zeros.data_ptr()
    return N.W4(codes.data_ptr(), scales.data_ptr(), zp, V, d, d // G, _DT[scales.dtype])


def _apart(t, name, *read):
    """Refuses an output that meets memory which the call reads: (tensor or None, what) each."""
    a0 = t.data_ptr()
    a1 = a0 + _extent(t)
    for r, what in read:
        if r is not None:
            p = r.data_ptr()
            if a0 < p + _extent(r) and p < a1:
                raise ValueError(f"{name} must not overlap {what}")


def _extent(t) -> int:
    """_span, at the price of a multiplication for contiguous tensors."""
    return t.nbytes if t.is_contiguous() else _span(t)


def _check_hidden_w4(hidden, w, dev):
    if hidden.dtype != torch.bfloat16:
        raise TypeError(f"hidden must be bfloat16, got {hidden.dtype}")
    _matrix(hidden, "hidden", dev, hidden.shape[0], w.d)
    B = hidden.shape[0]
    if not 1 <= B <= 256:
        raise ValueError(f"B={B} is outside [1, 256]")
    return B


@functools.lru_cache(maxsize=256)
def _w4_workspace_bytes(B: int, V: int, d: int, index: int) -> int:
    with torch.cuda.device(index):
        n = int(N.lib().mstar_lmhead_w4_workspace_bytes(B, V, d))
    if n <= 0:
        N.check(N.ERR_INVALID, "mstar_lmhead_w4_workspace_bytes")
    return n


def lmhead_w4_workspace(B: int, V: int, d: int, device) -> torch.Tensor:
    """Scratch for lmhead_logits_w4 calls of these sizes
    (mstar_lmhead_w4_workspace_bytes); calls that share it must not overlap."""
    dev = torch.device(device)
    index = torch.cuda.current_device() if dev.index is None else dev.index
    return torch.empty(_w4_workspace_bytes(B, V, d, index), dtype=torch.uint8, device=torch.device("cuda", index))


def lmhead_logits_w4(hidden: torch.Tensor, codes: torch.Tensor, scales: torch.Tensor, *, zeros=None,
                     out: torch.Tensor | None = None, dtype=torch.float32, status: torch.Tensor | None = None,
                     workspace: torch.Tensor | None = None) -> torch.Tensor:
    """hidden [B, d] (bfloat16, any row stride) times a 4-bit weight [V, d]
    transposed (mstar_lmhead_logits_w4): (code - zero) * scale, codes
    [V, d / 2] uint8 with the even column in the low four bits, scales
    [V, d / group] float32 or bfloat16, zeros uint8 of the same shape or None
    for 8.  fp32 sums, stored as float32 or bfloat16.  workspace: None takes
    fresh scratch from torch's allocator (safe on any stream and inside graph
    capture), or pass lmhead_w4_workspace's.  A bounded wait inside the kernel
    that runs out leaves wrong logits and sets bit 1 of `status`, and says so
    nowhere else: a caller that must know gives one and reads it."""
    w = _w4(codes, scales, zeros)
    dev = codes.device
    B = _check_hidden_w4(hidden, w, dev)
    if out is None:
        if dtype not in _DT:
            raise TypeError(f"dtype must be float32 or bfloat16, got {dtype}")
        out = torch.empty(B, w.V, dtype=dtype, device=dev)
    else:
        _matrix(out, "out", dev, B, w.V)
        _apart(out, "out", (hidden, "hidden"), (codes, "the codes"), (scales, "the scales"), (zeros, "the zeros"))
    if workspace is None:
        workspace = torch.empty(_w4_workspace_bytes(B, w.V, w.d, dev.index), dtype=torch.uint8, device=dev)
    wp, wn = _check_ws(workspace, dev)
    _call(dev, "mstar_lmhead_logits_w4", hidden.data_ptr(), _ld(hidden), B, ctypes.byref(w), out.data_ptr(),
          _DT[out.dtype], _ld(out), wp, wn, _status(status, dev))
    return out


def lmhead_step_w4(hidden: torch.Tensor, codes: torch.Tensor, scales: torch.Tensor, logits: torch.Tensor, *,
                   zeros=None, status=None, workspace: torch.Tensor | None = None, **kw) -> N.Params:
    """lmhead_logits_w4 into `logits` [B, V] (written) and one sampling step
    on it (mstar_sampler_lmhead_step_w4).  The sampling keywords are
    sampler_step's; the logits are read back from L2.  status: the head's, as
    for lmhead_logits_w4 (out_status is the sampling step's)."""
    w = _w4(codes, scales, zeros)
    dev = codes.device
    B = _check_hidden_w4(hidden, w, dev)
    _matrix(logits, "logits", dev, B, w.V)
    _apart(logits, "logits", (hidden, "hidden"), (codes, "the codes"), (scales, "the scales"), (zeros, "the zeros"))
    p = build_params(logits, **kw)
    if workspace is None:
        workspace = lmhead_w4_workspace(B, w.V, w.d, dev)
    wp, wn = _check_ws(workspace, dev)
    _call(dev, "mstar_sampler_lmhead_step_w4", ctypes.byref(p), hidden.data_ptr(), _ld(hidden), ctypes.byref(w), wp,
          wn, _status(status, dev))
    return p


def _ids_1d(ids, dev):
    if ids.dtype != torch.int64:
        raise TypeError(f"ids must be int64, got {ids.dtype}")
    if ids.device != dev:
        raise ValueError(f"ids must live on {dev}, got {ids.device}")
    if not ids.is_contiguous():
        raise ValueError("ids must be contiguous")
    return ids.numel()


def _lookup_out(ids, d, out, dtype, dev, *read):
    if out is None:
        if dtype not in _DT:
            raise TypeError(f"dtype must be float32 or bfloat16, got {dtype}")
        return torch.empty(*ids.shape, d, dtype=dtype, device=dev)
    if out.dtype not in _DT:
        raise TypeError(f"out must be float32 or bfloat16, got {out.dtype}")
    if out.device != dev or out.shape != (*ids.shape, d) or not out.is_contiguous():
        raise ValueError(f"out must be a contiguous {(*ids.shape, d)} tensor on {dev}")
    _apart(out, "out", *read)
    return out


def embed_tokens(ids: torch.Tensor, table: torch.Tensor, *, scale: float = 1.0, out: torch.Tensor | None = None,
                 dtype=None, status: torch.Tensor | None = None) -> torch.Tensor:
    """scale * table[ids] (mstar_embed_tokens): ids int64 of any shape, table
    [V, d] float32 or bfloat16 with contiguous rows; the result is ids.shape +
    (d,) of `dtype` (the table's by default).  The product is made in float32
    and rounded once.  A negative id gives zeros (a padding row); an id >= V
    does too and sets STATUS_BAD_ID in `status`."""
    dev = _cuda(table, "table")
    if table.dim() != 2:
        raise ValueError("table must be [V, d]")
    V, d = table.shape
    _matrix(table, "table", dev, V, d)
    n = _ids_1d(ids, dev)
    out = _lookup_out(ids, d, out, dtype or table.dtype, dev, (table, "the table"))
    st = _status(status, dev)
    if n:
        _call(dev, "mstar_embed_tokens", ids.data_ptr(), n, table.data_ptr(), _DT[table.dtype], V, d, _ld(table),
              scale, out.data_ptr(), _DT[out.dtype], st)
    return out


def embed_tokens_w4(ids: torch.Tensor, codes: torch.Tensor, scales: torch.Tensor, *, zeros=None, scale: float = 1.0,
                    out: torch.Tensor | None = None, dtype=torch.bfloat16,
                    status: torch.Tensor | None = None) -> torch.Tensor:
    """embed_tokens from a 4-bit table (mstar_embed_tokens_w4), the tied
    weight of lmhead_logits_w4: scale * (code - zero) * group scale."""
    w = _w4(codes, scales, zeros)
    dev = codes.device
    n = _ids_1d(ids, dev)
    out = _lookup_out(ids, w.d, out, dtype, dev, (codes, "the codes"), (scales, "the scales"), (zeros, "the zeros"))
    st = _status(status, dev)
    if n:
        _call(dev, "mstar_embed_tokens_w4", ids.data_ptr(), n, ctypes.byref(w), scale, out.data_ptr(), _DT[out.dtype],
              st)
    return out


@functools.lru_cache(maxsize=256)
def _embed_grad_workspace_bytes(n: int, V: int, d: int) -> int:
    nbytes = int(N.lib().mstar_embed_grad_workspace_bytes(n, V, d))
    if nbytes <= 0:
        raise ValueError(f"N={n}, V={V}, d={d} are outside [1, 2^24], [1, 2^21], [1, 65536]")
    return nbytes


def embed_tokens_grad(ids: torch.Tensor, dout: torch.Tensor, V: int, *, scale: float = 1.0,
                      base: torch.Tensor | None = None, out: torch.Tensor | None = None, dtype=None,
                      status: torch.Tensor | None = None) -> torch.Tensor:
    """The gradient of embed_tokens to its [V, d] table
    (mstar_embed_tokens_grad): base + scale * (the sum of dout's rows over the
    positions of each id), every row written.  dout is [N, d] (float32 or
    bfloat16, contiguous rows) for ids of N elements; base (None: zeros) has
    the result's type and may be `out` itself, which adds in place (the tied
    head's gradient, or an earlier micro-batch's).  Sums are float32 in
    position order, so equal inputs give equal bits; rounded once."""
    dev = _cuda(dout, "dout")
    n = _ids_1d(ids, dev)
    if dout.dim() != 2:
        raise ValueError("dout must be [N, d]")
    d = dout.shape[1]
    _matrix(dout, "dout", dev, n, d)
    if V < 1:
        raise ValueError("V must be >= 1")
    if out is None:
        out = torch.empty(V, d, dtype=dtype or (dout.dtype if base is None else base.dtype), device=dev)
    if base is not None:
        if base.dtype != out.dtype:
            raise TypeError(f"base must have out's type {out.dtype}, got {base.dtype}")
        _matrix(base, "base", dev, V, d)
        if not base.is_contiguous() or _overlap(base, out):
            raise ValueError("base must be contiguous, and out itself or apart from it")
    _matrix(out, "out", dev, V, d)
    if not out.is_contiguous():
        raise ValueError("out must be contiguous")
    if _overlap(dout, out) or out.data_ptr() == dout.data_ptr():
        raise ValueError("out must not overlap dout")
    st = _status(status, dev)
    if n == 0:
        if base is None:
            return out.zero_()
        return out if base.data_ptr() == out.data_ptr() else out.copy_(base)
    nbytes = _embed_grad_workspace_bytes(n, V, d)
    ws = torch.empty(nbytes, dtype=torch.uint8, device=dev)
    _call(dev, "mstar_embed_tokens_grad", ids.data_ptr(), n, dout.data_ptr(), _DT[dout.dtype], _ld(dout), V, d, scale,
          None if base is None else base.data_ptr(), out.data_ptr(), _DT[out.dtype], ws.data_ptr(), nbytes, st)
    return out


def _check_rows(logits, ids, temperature):
    dev = _cuda(logits, "logits")
    if logits.dim() != 2:
        raise ValueError("logits must be [N, V]")
    n, V = logits.shape
    _matrix(logits, "logits", dev, n, V)
    ip = _vec(ids, "ids", torch.int64, dev, n)
    if not 1e-5 <= temperature <= 1e5:
        raise ValueError(f"temperature must be in [1e-5, 1e5], got {temperature}")
    return dev, n, V, ip


def _grad_out(out, logits, dev, n, V, name):
    if out is None:
        return torch.empty(n, V, dtype=logits.dtype, device=dev)
    _matrix(out, name, dev, n, V)
    if out.dtype != logits.dtype:
        raise TypeError(f"{name} must have the logits' type {logits.dtype}, got {out.dtype}")
    if _overlap(out, logits):
        raise ValueError(f"{name} must be the logits themselves or apart from them")
    return out


def token_logprobs(logits: torch.Tensor, ids: torch.Tensor, *, temperature: float = 1.0,
                   logp: torch.Tensor | None = None, lse: torch.Tensor | None = None,
                   status: torch.Tensor | None = None):
    """(logp [N], lse [N]) float32 of ids [N] under softmax(logits /
    temperature), logits [N, V] float32 or bfloat16 (mstar_token_logprobs).
    -inf logits are masked ids; a row of nothing else gives -inf and
    STATUS_EMPTY.  A negative id is a padding row (logp 0); an id >= V counts
    as one and sets STATUS_BAD_ID."""
    dev, n, V, ip = _check_rows(logits, ids, temperature)
    if logp is None:
        logp = torch.empty(n, dtype=torch.float32, device=dev)
    if lse is None:
        lse = torch.empty(n, dtype=torch.float32, device=dev)
    lp, ls, st = _vec(logp, "logp", torch.float32, dev, n), _vec(lse, "lse", torch.float32, dev, n), _status(status, dev)
    if n:
        _call(dev, "mstar_token_logprobs", logits.data_ptr(), _DT[logits.dtype], n, V, _ld(logits), ip, temperature,
              lp, ls, st)
    return logp, lse


def token_logprobs_grad(logits: torch.Tensor, ids: torch.Tensor, lse: torch.Tensor, dlogp: torch.Tensor, *,
                        temperature: float = 1.0, out: torch.Tensor | None = None) -> torch.Tensor:
    """The gradient of sum(dlogp * logp) to the logits, of their type
    (mstar_token_logprobs_grad); lse is token_logprobs'.  out may be the
    logits themselves (replaced in place).  Padding and empty rows: zeros."""
    dev, n, V, ip = _check_rows(logits, ids, temperature)
    lp, dp = _vec(lse, "lse", torch.float32, dev, n), _vec(dlogp, "dlogp", torch.float32, dev, n)
    out = _grad_out(out, logits, dev, n, V, "out")
    if n:
        _call(dev, "mstar_token_logprobs_grad", logits.data_ptr(), _DT[logits.dtype], n, V, _ld(logits), ip,
              temperature, lp, dp, out.data_ptr(), _ld(out))
    return out


def policy_loss(logits: torch.Tensor, ids: torch.Tensor, old_logp: torch.Tensor | None, advantages: torch.Tensor, *,
                ref_logp: torch.Tensor | None = None, weights: torch.Tensor | None = None, temperature: float = 1.0,
                clip_low: float = 0.2, clip_high: float = 0.2, kl_coef: float = 0.0, grad: bool = True,
                loss: torch.Tensor | None = None, logp: torch.Tensor | None = None,
                dlogits: torch.Tensor | None = None, status: torch.Tensor | None = None):
    """Clipped policy loss per token and its gradient in one pass over the
    logits (mstar_policy_loss): (loss [N], logp [N], dlogits [N, V] or None).

        r = exp(logp - old_logp)           (old_logp None: on policy, r = 1)
        loss = -min(r A, clip(r, 1 - clip_low, 1 + clip_high) A)
               + kl_coef (exp(ref_logp - logp) - (ref_logp - logp) - 1)
        dlogits = the gradient of sum(weights * loss), weights None: 1

    logits [N, V] float32 or bfloat16; the per-token tensors are float32 [N].
    dlogits has the logits' type; give the logits themselves to replace them
    in place, or grad=False for the values alone.  A negative id is a padding
    row: loss 0, logp 0, a zero gradient, and its logits are not read."""
    dev, n, V, ip = _check_rows(logits, ids, temperature)
    f32 = torch.float32
    op, rp = _vec(old_logp, "old_logp", f32, dev, n), _vec(ref_logp, "ref_logp", f32, dev, n)
    ap, wp = _vec(advantages, "advantages", f32, dev, n), _vec(weights, "weights", f32, dev, n)
    if ap is None:
        raise ValueError("advantages must be given")
    if not (0 <= clip_low <= 1 and clip_high >= 0 and kl_coef >= 0):
        raise ValueError("clip_low must be in [0, 1], clip_high and kl_coef >= 0")
    if kl_coef > 0 and rp is None:
        raise ValueError("kl_coef needs ref_logp")
    if dlogits is not None and not grad:
        raise ValueError("dlogits is given, but grad is False")
    if loss is None:
        loss = torch.empty(n, dtype=f32, device=dev)
    if logp is None:
        logp = torch.empty(n, dtype=f32, device=dev)
    if grad:
        dlogits = _grad_out(dlogits, logits, dev, n, V, "dlogits")
    p = N.PolicyParams(logits.data_ptr(), _DT[logits.dtype], n, V, 0, _ld(logits), ip, op, rp, ap, wp, temperature,
                       clip_low, clip_high, kl_coef, _vec(loss, "loss", f32, dev, n), _vec(logp, "logp", f32, dev, n),
                       None, dlogits.data_ptr() if grad else None, _ld(dlogits) if grad else 0, _status(status, dev))
    if n:
        _call(dev, "mstar_policy_loss", ctypes.byref(p))
    return loss, logp, dlogits
