"""AdamW over a list of device tensors (snk_adamw_*), beside the model's own RMSProp.

Tensors are DeviceArrays (float32, float16, or uint16 holding bfloat16) or contiguous torch GPU
tensors; work on torch tensors runs on torch's current stream, work on DeviceArrays on the
library's. One launch covers every tensor, so a step costs the same few launches for ten tensors
or for hundreds.
"""
from __future__ import annotations

import ctypes as C
import operator
import struct

from . import _lib
from ._lib import DeviceView, call, f32, i64, vp


class AdamWCfg(C.Structure):
    """snk_adamw_cfg_t (struct_size set by the constructor: the library's ABI guard)"""
    _fields_ = [("struct_size", _lib.i32), ("param_dtype", _lib.i32), ("grad_dtype", _lib.i32), ("copy_dtype", _lib.i32),
                ("state_bits", _lib.i32), ("max_grad_norm", f32), ("beta1", _lib.f64), ("beta2", _lib.f64),
                ("eps", _lib.f64), ("seed", _lib.u64), ("reserved", i64)]

    def __init__(self, *args, **kw):
        super().__init__(C.sizeof(self), *args, **kw)


_dtype_of = operator.attrgetter("dtype")


def _same(buffers, what):
    kinds = {b.dtype for b in buffers}
    if len(kinds) != 1:
        raise ValueError(f"AdamW: the {what} must share one element type, got {sorted(kinds)}")
    kind = kinds.pop()
    if kind not in _lib.DTYPES:
        raise ValueError(f"AdamW: {what} of type {kind}")
    return _lib.DTYPES[kind]


class _Handle:
    """What a user's handle and a model's have in common."""

    _total = None
    _device = None   # the torch device of the tensors, None for DeviceArrays
    state_bits = 32

    @property
    def handle(self):
        return self._h

    @property
    def device(self):
        """Whose current stream the calls run on: the tensors' torch device, None for the library's own."""
        return self._device

    def _call(self, name, *args):
        _lib.call_on(self._device, name, *args)

    @property
    def steps(self) -> int:
        """Steps taken (waits for the stream). A skipped step is not counted. Assign to resume."""
        n = i64(0)
        self._call("snk_adamw_get_steps", self._h, C.byref(n))
        return n.value

    @steps.setter
    def steps(self, n: int) -> None:
        self._call("snk_adamw_set_steps", self._h, int(n))

    @property
    def total(self) -> int:
        """Places in the state layout: every tensor's size rounded up to 256."""
        if self._total is None:
            n = i64(0)
            call("snk_adamw_layout", self._h, C.byref(n), None)
            self._total = n.value
        return self._total

    @property
    def starts(self) -> list[int]:
        """Each tensor's first place in the state layout."""
        n, out = i64(0), (i64 * self._n)()
        call("snk_adamw_layout", self._h, C.byref(n), out)
        return list(out)

    def state(self) -> dict[str, DeviceView]:
        """The state's own device buffers, for checkpoints: m and v (float32, or the int8 / uint8
        codes with m_scale and v_scale, one a block of 256) and norm, the last step's gradient norm."""
        names = [("m", 0, "i1" if self.state_bits == 8 else "f4"), ("v", 1, "u1" if self.state_bits == 8 else "f4")]
        if self.state_bits == 8:
            names += [("m_scale", 2, "f4"), ("v_scale", 3, "f4")]
        out = {}
        for name, which, dt in names + [("norm", 4, "f4")]:
            p, n = vp(), i64(0)
            call("snk_adamw_state_ptr", self._h, which, C.byref(p), C.byref(n))
            out[name] = DeviceView(p.value, n.value // (1 if dt[1] == "1" else 4), dt, self)
        return out

    def reset(self) -> None:
        """Zero moments, step 0. Not while a graph is captured."""
        self.steps = 0   # first: refused under a capture, which is to record nothing then
        for name, view in self.state().items():
            if name != "norm" and view.nbytes:
                self._call("snk_memset", view.ptr, 0, view.nbytes)

    def moments(self, m=None, v=None) -> None:
        """The moments' values, written into m and v: [total] arrays of one type, either may be None,
        DeviceArrays or torch tensors as the parameters are (a model's: DeviceArrays)."""
        bufs = [None if x is None else _lib.device_buffer(x, "moments") for x in (m, v)]
        given = [b for b in bufs if b is not None]
        if not given:
            return
        for b in given:
            if b.size != self.total:
                raise ValueError(f"moments: {b.size} elements for {self.total} places")
        _lib.same_device(given, self._device)   # another kind's stream would not wait for the steps
        self._call("snk_adamw_moments", self._h, _same(given, "moments"), *[None if b is None else b.ptr for b in bufs])
        if self._device is not None:
            _lib.written([x for x in (m, v) if x is not None])


class AdamW(_Handle):
    """AdamW(params): every step(grads) names its gradients, a list of the parameters' length and sizes,
    new tensors each time if need be. AdamW(params, grads): step() uses these. params, grads (and
    copies) are kept alive and used at these addresses by every step until bind() names others (also where
    a tensor is given other memory, x.data = y: bind it again then).

    weight_decay: one number, or one per tensor. state_bits: 32, or 8 (codes in blocks of 256 with
    two fp32 scales each, v rounded stochastically with `seed`). max_grad_norm > 0 clips the global
    gradient norm and skips a step whose norm is not finite. copies: 16-bit tensors that receive the
    updated parameters too (fp32 master weights with bf16 working weights)."""

    def __init__(self, params, grads=None, *, lr: float = 1e-3, betas=(0.9, 0.999), eps: float = 1e-8, weight_decay=0.01,
                 state_bits: int = 32, max_grad_norm: float = 0.0, copies=None, seed: int = 0):
        keep = params, grads, copies = self._lists(params, grads, copies)
        ps, gs, cs = self._buffers(params, grads, copies)
        n = len(ps)
        wd = list(weight_decay) if isinstance(weight_decay, (list, tuple)) else [weight_decay] * n
        if len(wd) != n:
            raise ValueError(f"AdamW: {len(wd)} weight decays for {n} tensors")
        self.lr, self.state_bits, self._n = float(lr), int(state_bits), n
        self._sizes = [b.size for b in ps]
        self._types = self._types_of(ps, gs, cs)
        ptype, gtype, ctype = self._types
        cfg = AdamWCfg(ptype, max(gtype, 0), ctype, self.state_bits, float(max_grad_norm), float(betas[0]), float(betas[1]),
                       float(eps), int(seed), 0)
        self._device = ps[0].device
        self._pack = struct.Struct(f"={n}Q").pack   # a list of addresses
        h = vp()
        self._call("snk_adamw_create", C.byref(h), n, (i64 * n)(*self._sizes), (f32 * n)(*wd), C.byref(cfg))
        self._h = h
        self._bind(ps, gs, cs, keep)

    @staticmethod
    def _lists(*lists):   # of our own: what they hold has to live as long as its addresses are used
        return tuple(None if xs is None else tuple(xs) for xs in lists)

    @staticmethod
    def _buffers(params, grads, copies):
        lists = [[_lib.device_buffer(x, "AdamW") for x in xs or []] for xs in (params, grads, copies)]
        if not lists[0]:
            raise ValueError("AdamW: no tensors")
        for xs, other in ((grads, lists[1]), (copies or None, lists[2])):
            if xs is not None and [b.size for b in other] != [b.size for b in lists[0]]:
                raise ValueError("AdamW: params, grads (and copies) need the same sizes")
        _lib.same_device([b for bufs in lists for b in bufs])
        return lists

    @staticmethod
    def _types_of(ps, gs, cs):   # -1: none
        return _same(ps, "params"), _same(gs, "grads") if gs else -1, _same(cs, "copies") if cs else -1

    def _bind(self, ps, gs, cs, keep):
        n = self._n
        table = [(vp * n)(*[b.ptr for b in bufs]) if bufs else None for bufs in (ps, gs, cs)]
        self._call("snk_adamw_bind", self._h, *table)
        # aliases: a torch tensor's memory may be exchanged under it (x.data = y)
        self._keep = [[x.detach() if hasattr(x, "detach") else x for x in xs or ()] for xs in keep]
        if self._device is not None:
            # a tensor and its views count their changes together: one of each stands for all
            whole = [(x if x._base is None else x._base, y) for i in (0, 2) for x, y in zip(keep[i] or (), self._keep[i])]
            self._written = list({id(x): y for x, y in whole}.values())

    def bind(self, params, grads=None, copies=None) -> None:
        """Other addresses for the same tensors (moved parameters, other kept gradients), given as the
        constructor's were. Not while a graph is captured; graphs captured before use the new addresses
        from then on."""
        keep = params, grads, copies = self._lists(params, grads, copies)
        ps, gs, cs = self._buffers(params, grads, copies)
        if [b.size for b in ps] != self._sizes:
            raise ValueError("AdamW.bind: the sizes are those of the constructor")
        if self._types_of(ps, gs, cs) != self._types:
            raise ValueError("AdamW.bind: the element types, and which lists there are, are those of the constructor")
        _lib.same_device(ps, self._device)   # another kind's stream would not wait for the steps
        self._bind(ps, gs, cs, keep)

    def step(self, grads=None, *, lr: float | None = None, grad_scale: float = 1.0) -> None:
        """One step on these gradients, or the bound ones, times grad_scale (the inverse of a loss
        scale). Enqueued; nothing waits for it. A captured step keeps the gradients' addresses, lr and
        grad_scale, and needs this handle and the gradients as long as its graph is replayed."""
        lr = self.lr if lr is None else lr
        if grads is not None:
            if hasattr(grads, "data_ptr"):   # it would be taken apart
                raise TypeError("AdamW.step: a list of gradients, not a tensor")
            dtype, addresses = self._given(grads if isinstance(grads, (list, tuple)) else list(grads))
            self._call("snk_adamw_step_grads", self._h, dtype, self._pack(*addresses), lr, grad_scale)
        elif self._types[1] < 0:
            raise ValueError("AdamW.step: this handle was made without gradients, and none are given")
        else:
            self._call("snk_adamw_step", self._h, lr, grad_scale)
        if self._device is not None:
            _lib.written(self._written)

    def _given(self, grads):
        """(element type, addresses) of a step's own gradients. Torch's are looked at a property at a
        time, by C loops (a step on 261 tensors: 52 us of host time)."""
        if self._device is not None:
            tensor = _lib.torch_module().Tensor
            try:
                kinds = set(map(_dtype_of, grads))
                if len(kinds) == 1 and list(map(tensor.numel, grads)) == self._sizes and \
                        all(map(tensor.is_contiguous, grads)) and set(map(tensor.get_device, grads)) == {self._device.index}:
                    kind = _lib.DTYPES.get(_lib.TORCH_TYPES.get(kinds.pop()))
                    if kind is not None:
                        return kind, map(tensor.data_ptr, grads)
            except (AttributeError, TypeError):   # not all of them tensors
                pass
        bufs = [_lib.device_buffer(g, "AdamW.step") for g in grads]   # says what is wrong
        if [b.size for b in bufs] != self._sizes:
            raise ValueError("AdamW.step: the gradients need the parameters' sizes")
        _lib.same_device(bufs, self._device)
        return _same(bufs, "grads"), [b.ptr or 0 for b in bufs]

    def __del__(self):
        if getattr(self, "_h", None) and _lib._lib is not None:
            _lib._lib.snk_adamw_destroy(self._h)
            self._h = None


class ModelAdamW(_Handle):
    """The AdamW state of a DQNModel (DQNModel.use_adamw). The model owns it and its apply_grad and
    update step it; use_rmsprop or another use_adamw ends it, and its state()'s memory with it."""

    def __init__(self, model, handle, lr, state_bits, n):
        self._model, self._h, self._lr, self.state_bits, self._n = model, handle, float(lr), int(state_bits), int(n)

    @property
    def lr(self) -> float:
        """use_adamw's: another one takes another use_adamw."""
        return self._lr
