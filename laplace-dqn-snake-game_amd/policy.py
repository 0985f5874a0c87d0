"""Sampling from logits (snk_sample_logits) and the softmax policy over a Q-net's values, beside
epsilon_greedy (utils.jl:153-172).

Tensors are DeviceArrays or torch GPU tensors as in optim.py.
"""
from __future__ import annotations

import ctypes as C
import struct

import numpy as np

from . import _lib
from ._lib import DeviceArray, call, f32, i32, i64, vp


class SampleCfg(C.Structure):
    """snk_sample_cfg_t (struct_size set by the constructor: the library's ABI guard)"""
    _fields_ = [("struct_size", i32), ("dtype", i32), ("temperature", f32), ("top_k", i32), ("top_p", f32), ("min_p", f32),
                ("temperature_dev", vp), ("top_k_dev", vp), ("top_p_dev", vp), ("min_p_dev", vp)]

    def __init__(self, *args, **kw):
        super().__init__(C.sizeof(self), *args, **kw)


_CFG = struct.Struct("=iififfQQQQ")   # SampleCfg's bytes
_SETTINGS = (("temperature", "f32"), ("top_k", "i32"), ("top_p", "f32"), ("min_p", "f32"))
_NONE = (0, 0, 0, 0)


def _rows_of(x, b, what):
    """(rows, n, row stride in elements) of a 1-D or 2-D tensor whose rows are contiguous."""
    if len(b.shape) not in (1, 2):
        raise ValueError(f"{what}: {len(b.shape)} dimensions, expected [n] or [rows, n]")
    if len(b.shape) == 1:
        rows, n = 1, b.shape[0]
    else:
        rows, n = b.shape
    if b.device is None or x.is_contiguous():
        return rows, n, n
    st = x.stride()
    if n > 1 and st[-1] != 1:
        raise ValueError(f"{what}: the last dimension is not contiguous")
    return rows, n, st[0] if rows > 1 else n


def sample_logits(logits, u, *, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, mask=None, out=None, prob=None,
                  workspace=None):
    """One index per row of logits [rows, n] (or [n]), drawn with the given u [rows] in [0, 1).

    temperature, top_k, top_p and min_p (include/snakehip.h states the rules) are numbers or one
    value per row (float32, top_k int32). mask: bytes or bools [rows, n], non-zero forbids; [n] is for
    every row. A torch row stride of 0 (expand) shares one row. Returns out [rows] int32 (-1: nothing
    allowed), made here if not given; prob [rows] float32, if given, receives the probabilities.
    workspace: a uint8 tensor of sample_workspace(rows, n) bytes, made here if not given; calls in
    flight at the same time need one each."""
    b = _lib.device_buffer(logits, "logits", contiguous=False)
    device = b.device
    rows, n, ld = _rows_of(logits, b, "logits")
    dtype = _lib.DTYPES.get(b.dtype)
    if dtype is None:
        raise ValueError(f"logits: elements of type {b.dtype}")
    u_ptr = _lib.vector_ptr(u, "u", "f32", rows, device)
    m_ptr, ldm = None, n
    if mask is not None:
        mb = _lib.device_buffer(mask, "mask", contiguous=False)
        mrows, mn, ldm = _rows_of(mask, mb, "mask")
        if mb.dtype != "u8" or mn != n or mrows not in (1, rows):
            raise ValueError(f"mask: expected bytes [{rows}, {n}] or [{n}], got {mb.dtype} {list(mb.shape)}")
        if mrows == 1:
            ldm = 0
        _lib.same_device([mb], device)
        m_ptr = mb.ptr
    cfg = _cfg(dtype, [temperature, top_k, top_p, min_p], rows, device)
    made = out is None
    if made:
        out = _new(device, rows, np.int32)
    o_ptr = _lib.vector_ptr(out, "out", "i32", rows, device)
    p_ptr = None if prob is None else _lib.vector_ptr(prob, "prob", "f32", rows, device)
    w_ptr, w_bytes = None, 0
    need = sample_workspace(rows, n) if n > 4096 else 0
    if need:
        if workspace is None:
            workspace = _new(device, need, np.uint8)
        wb = _lib.device_buffer(workspace, "workspace")
        _lib.same_device([wb], device)
        w_ptr, w_bytes = wb.ptr, wb.size
    _lib.call_on(device, "snk_sample_logits", b.ptr, rows, n, ld, m_ptr, ldm, u_ptr, cfg, o_ptr, p_ptr, w_ptr, w_bytes)
    if device is not None and not (made and prob is None):
        _lib.written((prob,) if made else (out,) if prob is None else (out, prob))
    return out


def _cfg(dtype, settings, rows, device) -> bytes:
    """snk_sample_cfg_t of numbers, or of device tensors of a value a row."""
    arrays = _NONE
    for i, value in enumerate(settings):
        if value.__class__ is not float and not isinstance(value, (float, int, np.number)):
            what, kind = _SETTINGS[i]
            arrays = list(arrays)
            arrays[i] = _lib.vector_ptr(value, what, kind, rows, device)
            settings[i] = 0 if kind == "i32" else 1.0
    try:
        return _CFG.pack(_CFG.size, dtype, *settings, *arrays)
    except (struct.error, OverflowError) as e:
        raise ValueError(f"temperature, top_k, top_p, min_p = {settings}: {e}") from None


def sample_workspace(rows: int, n: int) -> int:
    """Bytes of workspace that sample_logits uses for rows x n logits (0: none)."""
    need = i64(0)
    call("snk_sample_workspace", rows, n, C.byref(need))
    return need.value


def _new(device, n, dtype):
    if device is None:
        return DeviceArray(n, dtype)
    torch = _lib.torch_module()
    return torch.empty(n, dtype=torch.int32 if dtype is np.int32 else torch.uint8, device=device)


def softmax_actions(game, model, *, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, seed: int = 0,
                    act: DeviceArray | None = None) -> np.ndarray:
    """Boltzmann exploration for every env, in epsilon_greedy's place: action indices drawn from
    softmax(Q / temperature) under the filters (numbers, or DeviceArrays of a value an env), with the
    counter RNG's u(seed, env, step). NaN among an env's Q values is action 0."""
    if act is not None:
        _lib.vector_ptr(act, "act", "u8", game.n_envs, None)
    else:
        act = DeviceArray(game.n_envs, np.uint8)
    cfg = _cfg(_lib.SNK_F32, [temperature, top_k, top_p, min_p], game.n_envs, None)
    call("snk_dqn_act_sample", model.handle, game.handle, cfg, int(seed), act.ptr)
    return act.numpy()
