"""The sampler's refusals that need no device, and its reference against counted cases (CPU)."""
import ctypes as C
import types

import numpy as np
import pytest

import sample_ref
import snake_amd
from snake_amd import _lib, policy
from snake_amd.policy import SampleCfg

ONE = 4096   # an address that is never read: every call below is refused before a launch


def _call(rows=1, n=8, ld=8, ldm=8, x=ONE, mask=None, u=ONE, idx=ONE, cfg=None, **change):
    base = dict(dtype=0, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0)
    cfg = SampleCfg(*{**base, **change}.values()) if cfg is None else cfg
    lib = snake_amd.load()
    st = lib.snk_sample_logits(x, rows, n, ld, mask, ldm, u, C.byref(cfg) if cfg else None, idx, None, None, 0)
    return st, lib.snk_last_error().decode()


@pytest.mark.parametrize("change,word", [
    (dict(dtype=7), "type"), (dict(temperature=-1.0), "temperature"), (dict(temperature=float("nan")), "temperature"),
    (dict(temperature=float("inf")), "temperature"), (dict(top_k=-1), "top_k"), (dict(top_p=1.5), "top_p"),
    (dict(top_p=-0.5), "top_p"), (dict(top_p=float("nan")), "top_p"), (dict(min_p=2.0), "min_p"),
    (dict(min_p=float("nan")), "min_p"), (dict(rows=-1), "rows"), (dict(rows=2 ** 31), "rows"), (dict(n=0), "logits a row"),
    (dict(n=2 ** 24 + 1, ld=2 ** 25), "logits a row"), (dict(ld=7), "ld"), (dict(ld=-8), "ld"),
    (dict(mask=ONE, ldm=3), "ld_mask"), (dict(x=None), "NULL"), (dict(u=None), "NULL"), (dict(idx=None), "NULL"),
    (dict(x=ONE + 2), "aligned"), (dict(x=ONE + 1, dtype=1), "aligned"), (dict(cfg=False), "cfg"),
])
def test_bad_calls_are_refused(change, word):
    st, msg = _call(**change)
    assert st == _lib.SNK_ERR_INVALID and word in msg, msg


def test_struct_size_guard():
    c = SampleCfg(0, 1.0, 0, 1.0, 0.0)
    assert C.sizeof(SampleCfg) == 56
    c.struct_size = 52
    st, msg = _call(cfg=c)
    assert st == _lib.SNK_ERR_INVALID and "struct_size" in msg
    assert snake_amd.load().snk_dqn_act_sample(None, None, C.byref(c), 0, None) == _lib.SNK_ERR_INVALID
    assert snake_amd.load().snk_sample_workspace(1, 1, None) == _lib.SNK_ERR_INVALID


def test_no_rows_is_no_work():
    assert _call(rows=0, x=None, u=None, idx=None)[0] == _lib.SNK_OK


def test_reference_on_counted_cases():
    x = np.log([1.0, 2.0, 4.0, 1.0])
    assert [sample_ref.row(x, u)[0] for u in (0.0, 0.124, 0.126, 0.374, 0.376, 0.874, 0.876)] == [0, 0, 1, 1, 2, 2, 3]
    assert sample_ref.row(x, 0.9, top_k=1)[:2] == (2, 1.0)
    assert sample_ref.row(x, 0.1, top_k=3)[0] == 0 and sample_ref.row(x, 0.99, top_k=3)[0] == 2    # the tie at 1: index 0
    assert sample_ref.row(x, 0.1, top_p=0.5)[0] == 2 and sample_ref.row(x, 0.1, top_p=0.51)[0] == 1
    assert sample_ref.row(x, 0.1, min_p=0.3)[0] == 1
    assert sample_ref.row(x, 0.999, mask=[0, 0, 1, 1])[0] == 1
    assert sample_ref.row(x, 0.5, temperature=0.0)[:2] == (2, 1.0)
    assert sample_ref.row([-np.inf, np.nan], 0.5, mask=[0, 1])[0] == -1
    assert sample_ref.row([1.0, np.inf, np.inf], 0.6)[:2] == (2, 0.5)


def _array(n, dtype):
    """A DeviceArray without memory: only its description is looked at."""
    a = object.__new__(snake_amd.DeviceArray)
    a.shape, a.dtype, a.ptr = (n,), np.dtype(dtype), _lib.vp(0)
    a.nbytes = n * a.dtype.itemsize
    return a


def test_actions_need_their_room(monkeypatch):
    """softmax_actions writes a byte an env: an array of another size or type is refused before any call."""
    def never(*args):
        raise AssertionError("called")
    monkeypatch.setattr(snake_amd.policy, "call", never)
    game = model = types.SimpleNamespace(n_envs=300, handle=None)
    for act in (_array(299, np.uint8), _array(301, np.uint8), _array(300, np.int32), _array(300, np.float32)):
        with pytest.raises(ValueError, match="act"):
            snake_amd.softmax_actions(game, model, act=act)
    with pytest.raises(TypeError):
        snake_amd.softmax_actions(game, model, act=np.zeros(300, np.uint8))


def test_settings_are_numbers_of_any_kind():
    """numpy's scalars are numbers; one that the library's types cannot hold is refused, not cut off."""
    want = policy._cfg(0, [0.5, 7, 0.75, 0.25], 3, None)
    assert want == bytes(SampleCfg(0, 0.5, 7, 0.75, 0.25, None, None, None, None))
    assert want == policy._cfg(0, [np.float32(0.5), np.int64(7), np.float64(0.75), np.float16(0.25)], 3, None)
    for bad in ([1.0, 2 ** 32 + 5, 1.0, 0.0], [1.0, -2 ** 31 - 1, 1.0, 0.0], [1.0, 5.5, 1.0, 0.0], [1e39, 0, 1.0, 0.0]):
        with pytest.raises(ValueError, match="temperature, top_k"):
            policy._cfg(0, bad, 3, None)


def test_actions_take_settings_of_each_env(monkeypatch):
    seen = []
    monkeypatch.setattr(policy, "call", lambda name, *args: seen.append((name, args)))
    game = model = types.SimpleNamespace(n_envs=300, handle=None)
    act = _array(300, np.uint8)
    act.numpy = lambda: None
    t = _array(300, np.float32)
    t.ptr = _lib.vp(8192)
    try:
        snake_amd.softmax_actions(game, model, temperature=t, top_k=2, act=act, seed=9)
        with pytest.raises(ValueError, match="top_k"):
            snake_amd.softmax_actions(game, model, top_k=t, act=act)
        with pytest.raises(ValueError, match="300"):
            snake_amd.softmax_actions(game, model, temperature=_array(299, np.float32), act=act)
        with pytest.raises(ValueError, match="top_k"):
            snake_amd.softmax_actions(game, model, top_k=2 ** 32 + 1, act=act)
    finally:
        t.ptr = None
    (name, args), = seen
    assert name == "snk_dqn_act_sample" and args[3] == 9
    assert args[2] == bytes(SampleCfg(0, 1.0, 2, 1.0, 0.0, 8192, None, None, None))
