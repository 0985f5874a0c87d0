"""AdamW's refusals that need no device, and its 64-bit reference against itself (CPU)."""
import ctypes as C

import numpy as np
import pytest

import adamw_ref
import snake_amd
from snake_amd import _lib
from snake_amd.optim import AdamWCfg

GOOD = dict(param_dtype=0, grad_dtype=0, copy_dtype=-1, state_bits=32, max_grad_norm=0.0, beta1=0.9, beta2=0.999,
            eps=1e-8, seed=0, reserved=0)


def _create(n=1, sizes=(8,), wd=(0.0,), cfg=None, **change):
    c = AdamWCfg(*{**GOOD, **change}.values()) if cfg is None else cfg
    h = _lib.vp()
    st = snake_amd.load().snk_adamw_create(C.byref(h), n, (C.c_int64 * len(sizes))(*sizes), (C.c_float * len(wd))(*wd),
                                           C.byref(c))
    return st, snake_amd.load().snk_last_error().decode()


@pytest.mark.parametrize("change,word", [
    (dict(param_dtype=3), "type"), (dict(grad_dtype=-1), "type"), (dict(copy_dtype=0), "copy_dtype"),
    (dict(state_bits=16), "state_bits"), (dict(beta1=1.0), "betas"), (dict(beta2=-0.1), "betas"),
    (dict(beta1=float("nan")), "betas"), (dict(eps=0.0), "eps"), (dict(eps=1e-60), "eps"), (dict(eps=float("inf")), "eps"),
    (dict(state_bits=8, eps=1e-13), "eps"), (dict(eps=2e30), "eps"), (dict(max_grad_norm=-1.0), "max_grad_norm"), (dict(max_grad_norm=float("nan")), "max_grad_norm"),
    (dict(reserved=1), "reserved"),
])
def test_bad_settings_are_refused(change, word):
    st, msg = _create(**change)
    assert st == _lib.SNK_ERR_INVALID and word in msg, msg


def test_bad_calls_are_refused():
    lib = snake_amd.load()
    bad = AdamWCfg(*GOOD.values())
    bad.struct_size = 60
    st, msg = _create(cfg=bad)
    assert st == _lib.SNK_ERR_INVALID and "struct_size" in msg
    assert C.sizeof(AdamWCfg) == 64
    assert _create(n=0)[0] == _lib.SNK_ERR_INVALID
    assert lib.snk_adamw_create(None, 1, None, None, None) == _lib.SNK_ERR_INVALID
    for name, args in (("snk_adamw_step", (None, 1.0, 1.0)), ("snk_adamw_bind", (None, None, None, None)),
                       ("snk_adamw_moments", (None, 0, None, None)), ("snk_adamw_get_steps", (None, None)),
                       ("snk_adamw_set_steps", (None, 1)), ("snk_adamw_layout", (None, None, None)),
                       ("snk_adamw_state_ptr", (None, 0, None, None)), ("snk_dqn_use_adamw", (None, None, 0.0, 0.0, None))):
        assert getattr(lib, name)(*args) == _lib.SNK_ERR_INVALID, name
    assert lib.snk_adamw_destroy(None) == _lib.SNK_OK
    assert lib.snk_swap_stream(None, 2, None, None) == _lib.SNK_ERR_INVALID


def test_host_tensors_are_refused():
    import torch
    with pytest.raises(ValueError, match="GPU"):
        snake_amd.AdamW([torch.zeros(4)], [torch.zeros(4)])
    with pytest.raises(TypeError):
        snake_amd.AdamW([np.zeros(4, np.float32)], [np.zeros(4, np.float32)])
    with pytest.raises(ValueError, match="no tensors"):
        snake_amd.AdamW([], [])


def test_stream_selection_is_exchanged():
    """snk_swap_stream keeps what snk_set_stream chose (no stream is used here)."""
    lib = snake_amd.load()
    old, given = _lib.vp(), C.c_int32(-1)
    assert lib.snk_swap_stream(_lib.vp(1234), 1, C.byref(old), C.byref(given)) == 0
    assert given.value == 0 and not old.value
    assert lib.snk_swap_stream(old, given.value, C.byref(old), C.byref(given)) == 0
    assert given.value == 1 and old.value == 1234
    assert lib.snk_swap_stream(None, 0, C.byref(old), C.byref(given)) == 0 and given.value == 0


def test_reference_codes_keep_the_mean():
    """The 8-bit rounding of v is unbiased: over all 65,536 random values the mean of the two
    neighbours' values is v to 2^-16 of their distance."""
    part = np.array([1e-9, 1e-4, 0.013, 0.5, 0.97, 1.0])
    low = np.minimum(np.floor(255 * part ** 0.25), 254)
    lo, hi = (low / 255) ** 4, ((low + 1) / 255) ** 4
    ups = np.ceil((part - lo) / (hi - lo) * 65536)   # the r in 0..65535 that go up
    mean = lo + (hi - lo) * np.minimum(ups, 65536) / 65536
    assert np.all(np.abs(mean - part) <= (hi - lo) / 65536 + 1e-15)


def test_reference_bits_are_the_counter_rng():
    import devrng
    seed, t = 0xABCDEF0123, 17
    got = adamw_ref.bits16(seed, t, 40)
    for i in (0, 1, 5, 39):
        assert got[i] == (devrng.rng_hash(seed, t, i // 4) >> (16 * (i % 4))) & 0xFFFF


def test_gradients_may_come_with_the_step():
    """AdamW(params) and step(grads): what is wrong with this call is the tensor, not the arguments."""
    import torch
    with pytest.raises(ValueError, match="GPU"):
        snake_amd.AdamW([torch.zeros(4)], lr=1e-3)
    lib, none = snake_amd.load(), (_lib.vp * 1)(None)
    assert lib.snk_adamw_step_grads(None, 0, none, 1.0, 1.0) == _lib.SNK_ERR_INVALID
    assert lib.snk_adamw_step_grads(_lib.vp(4096), 0, None, 1.0, 1.0) == _lib.SNK_ERR_INVALID   # before the handle is read


class _Owner(snake_amd.ModelAdamW):
    """A handle without a device: what it calls is recorded."""

    def __init__(self, device):
        self._h, self._device, self.state_bits, self._n = _lib.vp(4096), device, 32, 1


@pytest.fixture
def calls(monkeypatch):
    seen = []

    def call_on(device, name, *args):
        seen.append((device, name))
        if name == "snk_adamw_state_ptr":
            args[2]._obj.value, args[3]._obj.value = 8192, 16
    for module in (_lib, snake_amd.optim):
        monkeypatch.setattr(module, "call", lambda name, *args: call_on(None, name, *args))
    monkeypatch.setattr(_lib, "call_on", call_on)
    return seen


def test_state_is_reached_on_the_stream_of_the_steps(calls):
    """Memory that torch's streams order is read and written on torch's stream, the library's on its own."""
    for device in ("cuda:0", None):
        view = _Owner(device).state()["m"]
        del calls[:]
        view.numpy()
        view.upload(np.zeros(4))
        assert calls == [(device, "snk_memcpy_d2h"), (device, "snk_memcpy_h2d")]
        del calls[:]
        assert view.__cuda_array_interface__["data"] == (8192, False)
        assert calls == ([(None, "snk_synchronize")] if device is None else [])


def test_views_of_an_ended_state_are_refused(calls):
    opt = _Owner(None)
    view = opt.state()["m"]
    opt._h = None
    del calls[:]
    for use in (view.numpy, lambda: view.upload(np.zeros(4)), lambda: view.__cuda_array_interface__,
                lambda: _lib.device_buffer(view, "x")):
        with pytest.raises(ValueError, match="ended"):
            use()
    assert not calls


def test_a_model_s_rate_is_use_adamw_s():
    """Assigning would change nothing: the model holds the rate."""
    opt = snake_amd.ModelAdamW(None, _lib.vp(4096), 1e-3, 32, 10)
    assert opt.lr == 1e-3
    with pytest.raises(AttributeError):
        opt.lr = 1e-4
