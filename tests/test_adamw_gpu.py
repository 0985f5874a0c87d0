"""AdamW on the GPU against the 64-bit formula (adamw_ref: bounds that count fp32 roundings).

Every step is checked from the state the device itself held before it, so that bounds do not
accumulate; where a quantity is stored in fewer bits, half a step of that type is added.
"""
import ctypes as C

import numpy as np
import pytest

import adamw_ref as ref

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
TT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZES = [1, 3, 255, 256, 257, 0, 4095, 4096, 4097, 12289, 2]


def flat(tensors, sizes):
    starts, total = ref.places(sizes)
    out = np.zeros(total)
    for x, at, s in zip(tensors, starts, sizes):
        out[at:at + s] = x.double().cpu().numpy().reshape(-1)
    return out


def spread(values, sizes):
    starts, total = ref.places(sizes)
    out = np.zeros(total)
    for x, at, s in zip(values, starts, sizes):
        out[at:at + s] = x
    return out


def old_moments(opt):
    st = {k: x.numpy() for k, x in opt.state().items()}
    if opt.state_bits == 8:
        return ref.m_values(st["m"], st["m_scale"]), ref.v_values(st["v"], st["v_scale"]), st
    return st["m"].astype(np.float64), st["v"].astype(np.float64), st


def views(sizes, dtype, gen, std, offset):
    """Tensors cut out of one buffer with `offset` elements of canary before, between and after."""
    buf = torch.full((sum(sizes) + offset * (len(sizes) + 1),), 7.0, dtype=dtype, device="cuda")
    out, at = [], offset
    for s in sizes:
        buf[at:at + s] = (torch.randn(s, device="cuda", generator=gen) * std).to(dtype)
        out.append(buf[at:at + s])
        at += s + offset
    return buf, out


def canaries(buf, sizes, offset):
    keep, at = torch.ones_like(buf, dtype=torch.bool), offset
    for s in sizes:
        keep[at:at + s] = False
        at += s + offset
    return bool((buf[keep] == 7.0).all())


def check_step(opt, params, grads, sizes, wds, t, run, *, ptype, lr, b1, b2, eps, scale=1.0, max_norm=0.0, seed=0,
               copies=None):
    p, g = flat(params, sizes), flat(grads, sizes)
    m, v, _ = old_moments(opt)
    run()
    want = ref.Step(p, g, m, v, t, lr=lr, b1=b1, b2=b2, eps=eps, wd=spread(wds, sizes), scale=scale, max_norm=max_norm,
                    state_bits=opt.state_bits)
    got = flat(params, sizes)
    tol = want.ep + (ref.HALF[ptype] * (np.abs(want.p) + want.ep) + (2.0 ** -25 if ptype == "f16" else 0)
                     if ptype != "f32" else 0)
    assert np.all(np.abs(got - want.p) <= tol), float(np.max(np.abs(got - want.p) / np.maximum(tol, 1e-300)))
    m2, v2, st = old_moments(opt)
    if opt.state_bits == 8:
        want.codes_ok(st["m"], st["m_scale"], st["v"], st["v_scale"], ref.bits16(seed, t, m.size))
    else:
        assert np.all(np.abs(m2 - want.m) <= want.em) and np.all(np.abs(v2 - want.v) <= want.ev)
    if max_norm:
        assert abs(float(st["norm"][0]) - want.norm) <= 4 * ref.U * want.norm
    if copies is not None:
        c = flat(copies, sizes)
        assert np.all(np.abs(c - got) <= ref.HALF["bf16"] * np.abs(got))
    assert opt.steps == t


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("ptype,gtype", [("f32", "f32"), ("f32", "bf16"), ("bf16", "bf16"), ("f16", "f16"), ("bf16", "f32"),
                                         ("f32", "f16"), ("f16", "f32")])
@pytest.mark.parametrize("offset", [0, 1])
def test_steps_against_the_formula(snk, bits, ptype, gtype, offset):
    """Sizes around the block and chunk, aligned or not (offset 1: odd addresses), decay on some
    tensors only; steps without, under and over the norm limit."""
    gen = torch.Generator(device="cuda").manual_seed(bits + offset)
    pbuf, params = views(SIZES, TT[ptype], gen, 0.1, offset)
    gbuf, grads = views(SIZES, TT[gtype], gen, 0.02, offset)
    wds = [0.0 if i % 3 else 0.1 for i in range(len(SIZES))]
    hyper = dict(lr=1e-2, b1=0.9, b2=0.99, eps=1e-8)
    for max_norm in (0.0, 1.0, 100.0):
        opt = snk.AdamW(params, grads, lr=1e-2, betas=(0.9, 0.99), weight_decay=wds, state_bits=bits,
                        max_grad_norm=max_norm, seed=99)
        for t in (1, 2, 3):
            for g in grads:
                g.copy_((torch.randn(g.numel(), device="cuda", generator=gen) * 0.02 *
                         (torch.rand(g.numel(), device="cuda", generator=gen) > 0.3)).to(g.dtype))
            check_step(opt, params, grads, SIZES, wds, t, opt.step, ptype=ptype, max_norm=max_norm, seed=99, **hyper)
    assert canaries(pbuf, SIZES, offset) and canaries(gbuf, SIZES, offset)


@pytest.mark.parametrize("bits", [32, 8])
def test_wide_values(snk, bits):
    """Gradients over 40 orders of magnitude inside one block, large steps counts, other betas."""
    gen = torch.Generator(device="cuda").manual_seed(5)
    n = [1000]
    p = [torch.randn(1000, device="cuda", generator=gen)]
    g = [torch.randn(1000, device="cuda", generator=gen) * 10 ** (torch.rand(1000, device="cuda", generator=gen) * 24 - 18)]
    opt = snk.AdamW(p, g, lr=1e-3, betas=(0.5, 0.9), eps=1e-6, weight_decay=0.0, state_bits=bits, seed=3)
    opt.steps = 100000
    for t in (100001, 100002, 100003):
        check_step(opt, p, g, n, [0.0], t, opt.step, ptype="f32", lr=1e-3, b1=0.5, b2=0.9, eps=1e-6, seed=3)


def test_scaled_gradients_and_copies(snk):
    """fp32 master weights with bf16 copies; gradients of a loss scaled by 1024."""
    gen = torch.Generator(device="cuda").manual_seed(1)
    sizes = [777, 4096, 5]
    _, p = views(sizes, torch.float32, gen, 0.1, 3)
    _, g = views(sizes, torch.float16, gen, 3.0, 1)
    cbuf, c = views(sizes, torch.bfloat16, gen, 0.0, 1)
    opt = snk.AdamW(p, g, lr=1e-2, weight_decay=0.01, max_grad_norm=0.05, copies=c)
    for t in (1, 2):
        check_step(opt, p, g, sizes, [0.01] * 3, t, lambda: opt.step(grad_scale=1 / 1024), ptype="f32", lr=1e-2, b1=0.9,
                   b2=0.999, eps=1e-8, scale=1 / 1024, max_norm=0.05, copies=c)
    assert canaries(cbuf, sizes, 1)


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("bad", [float("inf"), float("-inf"), float("nan")])
def test_a_step_with_no_finite_norm_is_skipped(snk, bits, bad):
    p, g = torch.randn(5000, device="cuda"), torch.randn(5000, device="cuda")
    opt = snk.AdamW([p], [g], state_bits=bits, max_grad_norm=float("inf"))
    opt.step()
    before = [p.clone(), *[torch.as_tensor(x, device="cuda").clone() for k, x in opt.state().items() if k != "norm"]]
    assert opt.steps == 1
    g[4321] = bad
    opt.step()
    after = [p, *[torch.as_tensor(x, device="cuda") for k, x in opt.state().items() if k != "norm"]]
    assert opt.steps == 1 and all(torch.equal(a, b) for a, b in zip(before, after))
    assert not np.isfinite(opt.state()["norm"].numpy()[0])
    g[4321] = 0.5
    opt.step()
    assert opt.steps == 2 and not torch.equal(before[0], p)


def test_many_tensors(snk):
    """Over 128 tensors: the bind takes several launches, the step stays whole."""
    gen = torch.Generator(device="cuda").manual_seed(2)
    sizes = [(i * 37) % 700 for i in range(300)]
    _, p = views(sizes, torch.float32, gen, 0.1, 1)
    _, g = views(sizes, torch.float32, gen, 0.1, 1)
    wds = [0.01 * (i % 2) for i in range(300)]
    opt = snk.AdamW(p, g, weight_decay=wds, max_grad_norm=1.0)
    assert opt.starts == ref.places(sizes)[0] and opt.total == ref.places(sizes)[1]
    for t in (1, 2):
        check_step(opt, p, g, sizes, wds, t, opt.step, ptype="f32", lr=1e-3, b1=0.9, b2=0.999, eps=1e-8, max_norm=1.0)


@pytest.mark.parametrize("bits", [32, 8])
def test_equal_runs_are_equal_bit_for_bit(snk, bits):
    gen = torch.Generator(device="cuda").manual_seed(4)
    p0, g = torch.randn(3_000_001, device="cuda", generator=gen), torch.randn(3_000_001, device="cuda", generator=gen)
    out = []
    for _ in range(2):
        p = p0.clone()
        opt = snk.AdamW([p], [g], state_bits=bits, max_grad_norm=1.0, seed=8)
        for _ in range(3):
            opt.step()
        out.append([p, *[torch.as_tensor(x, device="cuda").clone() for x in opt.state().values()]])
    assert all(torch.equal(a, b) for a, b in zip(*out))


@pytest.mark.parametrize("bits", [32, 8])
def test_captured_step(snk, bits):
    """Replays of a captured step, with eager work and synchronisation between, equal eager steps."""
    gen = torch.Generator(device="cuda").manual_seed(6)
    p0 = torch.randn(70_001, device="cuda", generator=gen)
    gs = [torch.randn(70_001, device="cuda", generator=gen) for _ in range(5)]
    runs = []
    for captured in (False, True):
        p, g = p0.clone(), torch.zeros_like(p0)
        opt = snk.AdamW([p], [g], state_bits=bits, max_grad_norm=1.0, seed=1)
        if captured:
            graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.graph(graph, stream=side):
                opt.step()
        seen = []
        for i, x in enumerate(gs):
            g.copy_(x)
            graph.replay() if captured else opt.step()
            if i % 2:
                torch.cuda.synchronize()
            seen.append(p.clone())
            p.mul_(0.999)
        runs.append(seen)
        assert opt.steps == 5
    assert all(torch.equal(a, b) for a, b in zip(*runs))


def test_own_stream_and_device_arrays(snk):
    """DeviceArrays work on the library's stream; torch tensors on torch's current one."""
    rng = np.random.default_rng(0)
    p0, g0 = rng.standard_normal(5000).astype(np.float32), rng.standard_normal(5000).astype(np.float32)
    p, g = snk.DeviceArray.from_host(p0), snk.DeviceArray.from_host(g0)
    opt = snk.AdamW([p], [g], lr=1e-2, weight_decay=0.1)
    opt.step()
    side = torch.cuda.Stream()
    tp, tg = torch.from_numpy(p0).cuda(), torch.zeros(5000, device="cuda")
    topt = snk.AdamW([tp], [tg], lr=1e-2, weight_decay=0.1)
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        torch.cuda._sleep(20_000_000)       # the gradient arrives late on the side stream
        tg.copy_(torch.from_numpy(g0).pin_memory(), non_blocking=True)
        topt.step()
    side.synchronize()
    assert np.array_equal(p.numpy(), tp.cpu().numpy())


def test_rebinding(snk):
    p = [torch.ones(300, device="cuda")]
    a, b = [torch.full((300,), 1.0, device="cuda")], [torch.full((300,), -1.0, device="cuda")]
    opt = snk.AdamW(p, a, lr=0.1, betas=(0.0, 0.0), weight_decay=0.0)
    opt.step()
    assert torch.allclose(p[0], torch.full_like(p[0], 0.9), rtol=0, atol=1e-6)
    opt.bind(p, b)
    opt.step()
    assert torch.allclose(p[0], torch.full_like(p[0], 1.0), rtol=0, atol=1e-6)
    with pytest.raises(ValueError):
        opt.bind([torch.ones(301, device="cuda")], b)
    with pytest.raises(ValueError):
        opt.bind([x.half() for x in p], b)


def test_overlapping_tensors_are_refused(snk):
    x, g = torch.zeros(1000, device="cuda"), torch.zeros(1000, device="cuda")
    for params, grads in (([x[:500], x[499:999]], [g[:500], g[500:1000]]), ([x, x], [g, g]), ([x[:500]], [x[499:999]])):
        with pytest.raises(snk.SnakeHipError, match="overlaps"):
            snk.AdamW(params, grads)
    snk.AdamW([x[:500], x[500:]], [g[:500], g[:500]]).step()     # gradients may share memory
    c = torch.zeros(1000, dtype=torch.bfloat16, device="cuda")
    with pytest.raises(snk.SnakeHipError, match="overlaps"):
        snk.AdamW([x[:500], x[500:]], [g[:500], g[500:]], copies=[c[:500], c[400:900]])
    with pytest.raises(ValueError, match="contiguous"):
        snk.AdamW([x[::2]], [g[:500]])
    with pytest.raises(ValueError):
        snk.AdamW([x], [g[:999]])
    with pytest.raises(ValueError):
        snk.AdamW([x, c], [g, g])


def test_moments_values(snk):
    gen = torch.Generator(device="cuda").manual_seed(7)
    p, g = torch.zeros(1000, device="cuda"), torch.randn(1000, device="cuda", generator=gen)
    for bits in (32, 8):
        opt = snk.AdamW([p], [g], state_bits=bits)
        opt.step()
        m, v, _ = old_moments(opt)
        for dt in ("f32", "bf16", "f16"):
            out = [torch.full((opt.total,), 9.0, dtype=TT[dt], device="cuda") for _ in range(2)]
            opt.moments(*out)
            # fp32 values of codes: m 4 U; v 12 U, (b / 255) being 2 U off, squared 5 U, squared again
            # 11 U, times the scale 12 U
            for x, y, k in zip(out, (m, v), (4, 12)):
                assert np.all(np.abs(x.double().cpu().numpy() - y) <= (ref.HALF[dt] + k * ref.U) * np.abs(y) + 2.0 ** -25 * (dt == "f16"))
            opt.moments(out[0])
        with pytest.raises(ValueError):
            opt.moments(torch.zeros(7, device="cuda"))


def test_rounding_keeps_the_mean_of_v(snk):
    """v decays by 1 % a step with no gradient; nearest codes would never move. Over 400 blocks of
    one pattern the mean stays within five standard deviations of the exact decay: one step's rounding
    has at most a quarter of the squared code distance, (4 v / b)^2 / 4, as its variance."""
    blocks, steps = 400, 30
    g = torch.linspace(0.3, 1.0, 256, device="cuda").repeat(blocks)
    p = torch.zeros_like(g)
    opt = snk.AdamW([p], [g], lr=0.0, betas=(0.0, 0.99), weight_decay=0.0, state_bits=8, seed=11)
    opt.step()
    v = [torch.empty(opt.total, device="cuda") for _ in range(2)]
    opt.moments(*v)
    start = v[1].view(blocks, 256).double().mean(0)
    g.zero_()
    for _ in range(steps):
        opt.step()
    opt.moments(*v)
    got = v[1].view(blocks, 256).double().mean(0)
    want = start * 0.99 ** steps
    b = 255 * (want / want.max()) ** 0.25
    sd = (steps / blocks) ** 0.5 * 0.5 * 4 * start / b
    assert torch.all((got - want).abs() <= 5 * sd + 1e-5 * want), ((got - want).abs() / sd).max()


def test_offsets_past_32_bits(snk):
    n = 2 ** 31 + 777
    p = torch.zeros(n, dtype=torch.bfloat16, device="cuda")
    g = torch.zeros(n, dtype=torch.bfloat16, device="cuda")
    p[-1000:], g[-1000:] = 1.0, 0.5
    p[:1000], g[:1000] = 1.0, -0.5
    opt = snk.AdamW([p], [g], lr=0.25, betas=(0.0, 0.0), weight_decay=0.0, state_bits=8)
    opt.step()
    assert bool((p[-1000:] == 0.75).all()) and bool((p[:1000] == 1.25).all())
    assert not bool(p[1000:-1000].any())


# ------------------------------------------------------------------ the model's own update

def _replay(snk, n=256, bs=12):
    g = snk.SnakeGame(bs, 2, n_envs=n, autoreset=True)
    rb = snk.ReplayBuffer(4096, board_size=bs, n_frames=2)
    act = snk.DeviceArray(n, np.uint8)
    for _ in range(8):
        snk.synth_actions_dev(g, 5, act)
        snk.step_indices_dev(g, act.ptr, replay=rb)
    return g, rb


@pytest.mark.parametrize("deep", [False, True])
@pytest.mark.parametrize("bits", [32, 8])
def test_model_updates(snk, deep, bits):
    """apply_grad and update of a model on AdamW: parameters against the formula, weights decaying
    and biases not, and the forward pass that of the updated parameters."""
    _, rb = _replay(snk)
    m = snk.DQNModel(12, 3, n_frames=2, seed=3, deep=deep)
    start = m.get_params()
    opt = m.use_adamw(lr=1e-3, weight_decay=0.1, state_bits=bits, max_grad_norm=1.0, seed=21)
    perm = m.flux_index()
    sizes = ([576, 32, 9216, 32, 18432, 64, 147456, 64, 49 * 4096, 64, 192, 3] if deep else
             [288, 16, 4608, 32, 73728, 64, 49 * 4096, 64, 192, 3])
    assert sum(sizes) == m.P
    starts, total = ref.places(sizes)
    assert opt.starts == starts and opt.total == total
    ends = np.cumsum([0] + sizes)

    def layout(flux):
        packed = flux[perm].astype(np.float64)
        return spread([packed[a:b] for a, b in zip(ends, ends[1:])], sizes)

    wd = spread([0.1 if i % 2 == 0 else 0.0 for i in range(len(sizes))], sizes)
    for t in (1, 2, 3):
        idx, B = snk.sample(rb, seed=t)
        p, (mo, vo, _) = layout(m.get_params()), old_moments(opt)
        m.update(rb, idx, B)
        want = ref.Step(p, layout(m.grad), mo, vo, t, lr=1e-3, b1=0.9, b2=0.999, eps=1e-8, wd=wd, max_norm=1.0,
                        state_bits=bits)
        got = layout(m.get_params())
        assert np.all(np.abs(got - want.p) <= want.ep)
        assert opt.steps == t
    x = np.random.default_rng(0).integers(-1, 3, size=(5, 2, 144)).astype(np.float32)
    q = m(x)
    m.set_params(m.get_params())          # rebuilds the forward images
    assert np.array_equal(q, m(x)) and not np.array_equal(start, m.get_params())


def test_model_back_to_rmsprop(snk):
    _, rb = _replay(snk)
    a, b = (snk.DQNModel(12, 3, n_frames=2, seed=3) for _ in range(2))
    idx, B = snk.sample(rb, seed=1)
    for m in (a, b):
        m.update(rb, idx, B)
    opt = a.use_adamw(lr=0.0)
    with pytest.raises(snk.SnakeHipError, match="belongs"):
        snk._lib.call("snk_adamw_step", opt.handle, 0.1, 1.0)
    with pytest.raises(snk.SnakeHipError, match="belongs"):
        snk._lib.call("snk_adamw_destroy", opt.handle)
    a.use_rmsprop()
    with pytest.raises(snk.SnakeHipError):
        opt.steps
    for m in (a, b):
        m.update(rb, idx, B)
    assert np.array_equal(a.get_params(), b.get_params())
    assert np.array_equal(a.get_params(snk.SNK_NET_OPT_STATE), b.get_params(snk.SNK_NET_OPT_STATE))
    with pytest.raises(snk.SnakeHipError):
        a.use_adamw(lr=float("nan"))


@pytest.mark.parametrize("deep", [False, True])
def test_trainer_on_adamw(snk, deep):
    """Captured training iterations equal eager ones bit for bit; two updates an iteration; the
    optimizer may change between runs (graphs are captured again)."""
    out = []
    for graph in (True, False):
        model = snk.DQNModel(12, 3, n_frames=2, seed=5, deep=deep)
        opt = model.use_adamw(lr=1e-3, weight_decay=0.01, max_grad_norm=10.0, state_bits=8, seed=2)
        tr = snk.Trainer(model=model, game=snk.SnakeGame(12, 2, n_envs=64, autoreset=True), capacity=2048,
                         updates_per_iter=2, target_update_rate=4, seed=9, graph_unroll=4)
        snk.fill_buffer_(tr, graph=graph)
        tr.run(10, graph=graph)
        assert opt.steps == 20 and tr.stats()["updates"] == 20
        got = [model.get_params(), model.get_params(snk.SNK_NET_TARGET), tr.losses]
        model.use_rmsprop()
        tr.run(5, graph=graph)
        got.append(model.get_params())
        out.append(got)
    assert all(np.array_equal(a, b) for a, b in zip(*out))
    assert np.all(np.isfinite(out[0][0]))


def test_lists_of_the_caller_may_change(snk):
    """Generators are taken, and what the caller's lists lose later is kept."""
    gen = torch.Generator(device="cuda").manual_seed(21)
    ps = [torch.randn(5000, device="cuda", generator=gen) for _ in range(3)]
    gs = [torch.randn(5000, device="cuda", generator=gen) for _ in range(3)]
    want = [p.clone() for p in ps]
    same = snk.AdamW(want, [g.clone() for g in gs])
    opt = snk.AdamW((p for p in ps), gs)
    del gs[:]
    others = [torch.full((5000,), 7.0, device="cuda") for _ in range(12)]   # may take freed places
    same.step()
    opt.step()
    assert all(torch.equal(a, b) for a, b in zip(ps, want))
    assert all(bool((x == 7.0).all()) for x in others)


def test_refused_under_capture(snk):
    """A handle is made and tensors are bound outside a capture; the capture goes on."""
    p, g, q = (torch.ones(300, device="cuda") for _ in range(3))
    opt = snk.AdamW([p], [g])
    model = snk.DQNModel(12, 3, n_frames=2)
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.graph(graph, stream=side):
        with pytest.raises(snk.SnakeHipError, match="captured"):
            snk.AdamW([q], [g])
        with pytest.raises(snk.SnakeHipError, match="captured"):
            opt.bind([q], [g])
        opt.step()
    assert opt.steps == 0
    graph.replay()
    torch.cuda.synchronize()
    assert opt.steps == 1 and bool((p < 1).all()) and bool((q == 1).all())
    assert model.use_adamw().steps == 0


def test_moments_into_one_array_are_refused(snk):
    p, g = torch.ones(300, device="cuda"), torch.ones(300, device="cuda")
    opt = snk.AdamW([p], [g])
    x = torch.empty(opt.total, device="cuda")
    with pytest.raises(snk.SnakeHipError, match="one array"):
        opt.moments(x, x)


@pytest.mark.parametrize("bits", [32, 8])
def test_reset_optimizer(snk, bits):
    """reset() and DQNModel.reset_optimizer start the optimizer in force again, the state object lost or not."""
    model = snk.DQNModel(12, 3, n_frames=2, seed=3)
    assert model.adamw is None
    opt = model.use_adamw(lr=1e-3, state_bits=bits)
    assert model.adamw is opt
    gen = np.random.default_rng(1)
    start, grad = model.get_params(), gen.standard_normal(model.P).astype(np.float32)

    def step():
        model.set_params(start)
        model.set_params(grad, snk.SNK_NET_GRAD)
        model.apply_grad()
        return model.get_params()

    first, second = step(), step()
    assert not np.array_equal(first, second)
    opt.reset()
    assert opt.steps == 0 and not opt.state()["m"].numpy().any()
    assert np.array_equal(step(), first)
    del opt
    model.reset_optimizer()
    assert model.adamw.steps == 0
    assert np.array_equal(step(), first)
    model.use_rmsprop()
    assert model.adamw is None
    first, second = step(), step()
    model.reset_optimizer()
    assert np.array_equal(step(), first) and not np.array_equal(first, second)


def test_more_elements_than_one_grid(snk):
    """Places past 2^34: the tail of a tensor moves as a small tensor of its own does."""
    big, tail = (1 << 34) + 1000, 3048   # the tail starts on a block
    if torch.cuda.mem_get_info()[0] < 140 << 30:
        pytest.skip("needs 140 GB of free memory")
    gen = torch.Generator(device="cuda").manual_seed(4)
    p, g = (torch.zeros(big, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    p[-tail:] = torch.randn(tail, device="cuda", generator=gen)
    g[-tail:] = torch.randn(tail, device="cuda", generator=gen)
    p2, g2 = p[-tail:].clone(), g[-tail:].clone()
    a = snk.AdamW([p], [g], state_bits=8, lr=1e-2)
    b = snk.AdamW([p2], [g2], state_bits=8, lr=1e-2)
    a.step()
    b.step()
    assert torch.equal(p[-tail:], p2) and not bool(p[:1 << 20].any())
    x, y = a.state(), b.state()
    for name in ("m", "m_scale", "v_scale"):
        small = torch.as_tensor(y[name], device="cuda")
        assert torch.equal(torch.as_tensor(x[name], device="cuda")[-small.numel():], small), name
    assert a.steps == 1
    del a, p, g
    torch.cuda.empty_cache()


def test_moments_of_the_parameters_kind(snk):
    """DeviceArrays are written on the library's stream, torch tensors on torch's: they are not mixed."""
    p, g = torch.ones(300, device="cuda"), torch.ones(300, device="cuda")
    opt = snk.AdamW([p], [g])
    with pytest.raises(ValueError, match="mix"):
        opt.moments(snk.DeviceArray(opt.total, np.float32))
    held = snk.DQNModel(12, 3, n_frames=2).use_adamw()
    with pytest.raises(ValueError, match="mix"):
        held.moments(torch.empty(held.total, device="cuda"))
    out = snk.DeviceArray(held.total, np.float32)
    held.moments(out)
    assert not out.numpy().any()


@pytest.mark.parametrize("param,grad,bits,copies,n", [
    ("f32", "bf16", 32, "f16", 25_000_003), ("f32", "f32", 32, None, 25_000_003), ("bf16", "f32", 32, None, 25_000_003),
    ("f16", "f16", 32, None, 30_000_001), ("bf16", "bf16", 8, None, 57_000_001), ("f32", "f16", 8, "bf16", 45_000_001),
    ("f16", "f32", 8, None, 45_000_001)])
def test_large_steps(snk, param, grad, bits, copies, n):
    """More bytes than the caches hold take the accesses past them: the same bits as the halves, stepped
    by handles of their own, get (but for v's codes, whose rounding goes by the place)."""
    gen = torch.Generator(device="cuda").manual_seed(n)
    sizes = [n // 2 - 5, n - n // 2 + 5]
    pb, ps = views(sizes, TT[param], gen, 0.1, 3)
    gb, gs = views(sizes, TT[grad], gen, 0.01, 1)
    cs = None if copies is None else [torch.zeros(s, dtype=TT[copies], device="cuda") for s in sizes]
    halves = [[p.clone(), g.clone(), None if cs is None else torch.zeros_like(cs[i])] for i, (p, g) in enumerate(zip(ps, gs))]
    how = dict(state_bits=bits, lr=1e-2, weight_decay=0.1, seed=3)
    opt = snk.AdamW(ps, gs, copies=cs, **how)
    opts = [snk.AdamW([p], [g], copies=None if c is None else [c], **how) for p, g, c in halves]
    for steps in range(2 if bits == 32 else 1):
        opt.step()
        for o in opts:
            o.step()
    st = {k: torch.as_tensor(x, device="cuda") for k, x in opt.state().items()}
    for i, (half, o) in enumerate(zip(halves, opts)):
        assert torch.equal(ps[i], half[0])
        assert cs is None or torch.equal(cs[i], half[2])
        for k, x in o.state().items():
            x = torch.as_tensor(x, device="cuda")
            at = opt.starts[i] // (256 if "scale" in k else 1)
            if k != "norm" and (k != "v" or bits == 32):
                assert torch.equal(st[k][at:at + x.numel()], x), k
    assert canaries(pb, sizes, 3) and canaries(gb, sizes, 1)


# ------------------------------------------------------------------ gradients that come with the step

@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("ptype,gtype", [("f32", "f32"), ("f32", "bf16"), ("bf16", "f32"), ("f16", "f16")])
def test_gradients_with_the_step(snk, bits, ptype, gtype):
    """New tensors every step, at odd addresses too: the formula, and the bits of bound gradients."""
    gen = torch.Generator(device="cuda").manual_seed(bits)
    for max_norm in (0.0, 1.0):
        pbuf, params = views(SIZES, TT[ptype], gen, 0.1, 1)
        twins = [p.clone() for p in params]
        opt = snk.AdamW(params, lr=1e-2, betas=(0.9, 0.99), weight_decay=0.1, state_bits=bits, max_grad_norm=max_norm, seed=99)
        held = [torch.zeros(s, dtype=TT[gtype], device="cuda") for s in SIZES]
        twin = snk.AdamW(twins, held, lr=1e-2, betas=(0.9, 0.99), weight_decay=0.1, state_bits=bits, max_grad_norm=max_norm,
                         seed=99)
        for t in (1, 2, 3):
            gbuf, grads = views(SIZES, TT[gtype], gen, 0.02, t % 2)
            for a, b in zip(held, grads):
                a.copy_(b)
            check_step(opt, params, grads, SIZES, [0.1] * len(SIZES), t, lambda: opt.step(grads), ptype=ptype, lr=1e-2, b1=0.9,
                       b2=0.99, eps=1e-8, max_norm=max_norm, seed=99)
            twin.step()
            assert canaries(gbuf, SIZES, t % 2)
        assert canaries(pbuf, SIZES, 1) and all(torch.equal(a, b) for a, b in zip(params, twins))


@pytest.mark.parametrize("max_norm", [0.0, 1.0])
def test_many_gradients_with_the_step(snk, max_norm):
    """Over 384 tensors: their addresses take several launches; a generator, scaled, with copies."""
    gen = torch.Generator(device="cuda").manual_seed(2)
    sizes = [(i * 37) % 700 for i in range(800)]
    _, p = views(sizes, torch.float32, gen, 0.1, 1)
    _, c = views(sizes, torch.bfloat16, gen, 0.0, 1)
    opt = snk.AdamW(p, weight_decay=0.01, max_grad_norm=max_norm, copies=c)
    for t in (1, 2):
        _, g = views(sizes, torch.float16, gen, 3.0, t)
        check_step(opt, p, g, sizes, [0.01] * 800, t, lambda: opt.step((x for x in g), lr=1e-2, grad_scale=0.125), ptype="f32",
                   lr=1e-2, b1=0.9, b2=0.999, eps=1e-8, scale=0.125, max_norm=max_norm, copies=c)


def test_bound_gradients_stay(snk):
    """step(grads), of another type too, leaves what is bound."""
    p = torch.ones(3000, device="cuda")
    bound, own = torch.full((3000,), 1.0, device="cuda"), torch.full((3000,), -1.0, device="cuda", dtype=torch.bfloat16)
    opt = snk.AdamW([p], [bound], lr=0.125, betas=(0.0, 0.0), weight_decay=0.0)
    for call, want in ((lambda: opt.step(), 0.875), (lambda: opt.step([own]), 1.0), (lambda: opt.step(), 0.875)):
        call()
        assert torch.allclose(p, torch.full_like(p, want), rtol=0, atol=1e-6)


@pytest.mark.parametrize("max_norm", [0.0, 1.0])
def test_captured_steps_with_gradients(snk, max_norm):
    """Two captured steps on gradients of their own, replayed in turn with eager steps on others between."""
    gen = torch.Generator(device="cuda").manual_seed(6)
    p0 = torch.randn(70_001, device="cuda", generator=gen)
    runs = []
    for captured in (False, True):
        gen = torch.Generator(device="cuda").manual_seed(7)
        p = p0.clone()
        gs = [torch.zeros_like(p0) for _ in range(2)]
        opt = snk.AdamW([p], state_bits=8, max_grad_norm=max_norm, seed=1)
        graphs = []
        if captured:
            side = torch.cuda.Stream()
            side.wait_stream(torch.cuda.current_stream())
            for g in gs:
                graphs.append(torch.cuda.CUDAGraph())
                with torch.cuda.graph(graphs[-1], stream=side):
                    opt.step([g])
        seen = []
        for i in range(6):
            for j, g in enumerate(gs):
                g.copy_(torch.randn(70_001, device="cuda", generator=gen))
                graphs[j].replay() if captured else opt.step([g])
                seen.append(p.clone())
            if i % 2:
                opt.step([torch.randn(70_001, device="cuda", generator=gen).bfloat16()])
                torch.cuda.synchronize()
        assert opt.steps == 15
        runs.append(seen)
    assert all(torch.equal(a, b) for a, b in zip(*runs))


def test_gradients_of_device_arrays(snk):
    rng = np.random.default_rng(0)
    p0, g0 = rng.standard_normal(5000).astype(np.float32), rng.standard_normal(5000).astype(np.float32)
    p, t = snk.DeviceArray.from_host(p0), torch.from_numpy(p0).cuda()
    opt, twin = snk.AdamW([p]), snk.AdamW([t])
    opt.step([snk.DeviceArray.from_host(g0)])
    twin.step([torch.from_numpy(g0).cuda()])
    assert np.array_equal(p.numpy(), t.cpu().numpy())


def test_refused_gradients(snk):
    """Each refused call leaves parameters and count as they were."""
    x = torch.ones(1000, device="cuda")
    p, g = [x[:300], x[400:900]], [torch.ones(300, device="cuda"), torch.ones(500, device="cuda")]
    opt = snk.AdamW(p)
    for bad, error, word in ((None, ValueError, "without gradients"), (g[0], TypeError, "a list"), (0.1, TypeError, "iterable"), (g[:1], ValueError, "sizes"), (g[::-1], ValueError, "sizes"),
                             ([g[0], None], TypeError, "neither"), ([g[0], g[1].half()], ValueError, "one element type"),
                             ([a.int() for a in g], ValueError, "i32"), ([a.double() for a in g], ValueError, "float64"),
                             ([a.cpu() for a in g], ValueError, "GPU"), ([], ValueError, "sizes"),
                             ([g[0], torch.ones(1000, device="cuda")[::2]], ValueError, "contiguous"),
                             ([g[0], snk.DeviceArray(500, np.float32)], ValueError, "mix"),
                             ([g[0], x[:500]], snk.SnakeHipError, "overlaps"), ([x[600:900], g[1]], snk.SnakeHipError, "overlaps"),
                             ([x[301:601], g[1]], snk.SnakeHipError, "overlaps"), ([x[100:400], g[1]], snk.SnakeHipError, "overlaps")):
        with pytest.raises(error, match=word):
            opt.step(bad)
    with pytest.raises(ValueError, match="constructor"):
        opt.bind(p, g)
    assert opt.steps == 0 and bool((x == 1).all())
    opt.bind(p[:1] + [x[500:1000]])
    opt.step(g)
    assert opt.steps == 1 and bool((x[:300] < 1).all()) and bool((x[300:500] == 1).all()) and bool((x[500:] < 1).all())
    with pytest.raises(snk.SnakeHipError, match="belongs"):
        held = snk.DQNModel(12, 3, n_frames=2).use_adamw()
        snk._lib.call("snk_adamw_step_grads", held.handle, 0, (C.c_void_p * 10)(), 0.1, 1.0)


def test_state_after_a_late_step(snk):
    """The state is read after a step that is still to run on torch's stream, and written after it too."""
    p, g = torch.zeros(1000, device="cuda"), torch.zeros(1000, device="cuda")
    opt = snk.AdamW([p], [g], betas=(0.0, 0.0))
    torch.cuda.synchronize()
    with torch.cuda.stream(torch.cuda.Stream()):
        for value in (3.0, 5.0):
            torch.cuda._sleep(20_000_000)
            g.fill_(value)
            opt.step()
            assert np.all(opt.state()["m"].numpy()[:1000] == value)
        torch.cuda._sleep(20_000_000)
        opt.step()
        opt.state()["m"].upload(np.full(opt.total, 9.0, np.float32))
        assert np.all(opt.state()["m"].numpy() == 9.0)
        torch.cuda.current_stream().synchronize()


def test_torch_gets_a_model_s_finished_state(snk):
    model = snk.DQNModel(12, 3, n_frames=2, seed=3)
    opt = model.use_adamw(lr=1e-3, betas=(0.0, 0.9))
    model.set_params(np.full(model.P, 0.5, np.float32), snk.SNK_NET_GRAD)
    for _ in range(50):
        model.apply_grad()
    m = torch.as_tensor(opt.state()["m"], device="cuda")
    assert int((m == 0.5).sum()) == model.P
    view = opt.state()["m"]
    model.use_rmsprop()
    with pytest.raises(ValueError, match="ended"):
        view.numpy()


@pytest.mark.parametrize("bad", [float("inf"), float("-inf"), float("nan")])
def test_a_lost_element_is_lost_alone(snk, bad):
    """Without a norm pass an infinite gradient takes one parameter with it; its block's 255 others, whose
    8-bit scales it must not reach, move as they do beside a gradient of 0."""
    gen = torch.Generator(device="cuda").manual_seed(3)
    p0, g = torch.randn(2000, device="cuda", generator=gen), torch.randn(2000, device="cuda", generator=gen)
    at, out = 777, []
    for value in (0.0, bad):
        p = p0.clone()
        opt = snk.AdamW([p], state_bits=8, seed=5)
        for t in range(4):
            h = g * (1 + t)
            h[at] = value if t == 1 else 0.0
            opt.step([h])
        st = {k: x.numpy() for k, x in opt.state().items()}
        assert np.all(np.isfinite(st["m_scale"])) and np.all(np.isfinite(st["v_scale"]))
        st["m"][at] = st["v"][at] = 0
        out.append((p, st))
    assert bool(torch.isnan(out[1][0][at]))
    rest = torch.arange(2000, device="cuda") != at
    assert torch.equal(out[0][0][rest], out[1][0][rest])
    for k in ("m", "v", "m_scale", "v_scale"):
        assert np.array_equal(out[0][1][k], out[1][1][k]), k


@pytest.mark.parametrize("max_norm", [0.0, float("inf")])
@pytest.mark.parametrize("bits", [32, 8])
def test_a_square_past_fp32(snk, bits, max_norm):
    """A finite gradient whose square is not: the norm lets it pass, nothing becomes infinite or NaN, and the
    parameter takes no step by a second moment that is out of range. (An 8-bit block's other v
    become the first code of a very large scale: those parameters stand still, finite.)"""
    p0 = torch.randn(1000, device="cuda", generator=torch.Generator(device="cuda").manual_seed(3))
    p, g = p0.clone(), torch.full((1000,), 0.5, device="cuda")
    opt = snk.AdamW([p], [g], lr=1e-2, weight_decay=0.0, state_bits=bits, max_grad_norm=max_norm)
    for t in range(5):
        g[300] = 2e19 if t == 1 else -1e-3
        opt.step()
        if t == 1:
            before = p[300].clone()
        if t > 1:
            assert torch.equal(p[300], before)   # v / (1 - b2^t) is infinite in these steps
    assert bool(torch.isfinite(p).all()) and opt.steps == 5
    far = torch.arange(1000, device="cuda") >= 512          # other blocks
    q = p0.clone()
    twin = snk.AdamW([q], [torch.full((1000,), 0.5, device="cuda")], lr=1e-2, weight_decay=0.0, state_bits=bits)
    for t in range(5):
        twin.step()
    assert torch.equal(p[far], q[far])
    if bits == 8:
        st = opt.state()
        assert np.all(np.isfinite(st["m_scale"].numpy())) and np.all(np.isfinite(st["v_scale"].numpy()))


def test_binding_of_another_kind_is_refused(snk):
    """A handle's calls stay on one stream: torch tensors and DeviceArrays do not follow one another, and a
    refused bind changes nothing."""
    p, g, q = (torch.ones(300, device="cuda") for _ in range(3))
    a, b = (snk.DeviceArray.from_host(np.ones(300, np.float32)) for _ in range(2))
    opt, own = snk.AdamW([p], [g]), snk.AdamW([a], [b])
    with pytest.raises(ValueError, match="mix"):
        opt.bind([a], [b])
    with pytest.raises(ValueError, match="mix"):
        own.bind([q], [g])
    with pytest.raises(snk.SnakeHipError, match="overlaps"):
        opt.bind([q], [q])
    assert opt.device == p.device and own.device is None
    opt.step()
    own.step()
    assert opt.steps == own.steps == 1 and bool((q == 1).all())
    assert np.array_equal(p.cpu().numpy(), a.numpy()) and bool((p < 1).all())


def test_exchanged_memory_is_kept(snk):
    """x.data = y takes a parameter's memory away; the handle's steps go on there and nowhere else."""
    p, g = torch.nn.Parameter(torch.ones(5000, device="cuda")), torch.ones(5000, device="cuda")
    old = [p.data_ptr(), g.data_ptr()]
    opt = snk.AdamW([p], [g], lr=0.125, betas=(0.0, 0.0), weight_decay=0.0)
    p.data, g.data = (torch.full((5000,), 7.0, device="cuda") for _ in range(2))
    others = [torch.full((5000,), 7.0, device="cuda") for _ in range(12)]   # would take freed places
    assert not {x.data_ptr() for x in others + [p, g]} & set(old)
    opt.step()
    assert opt.steps == 1 and all(bool((x == 7.0).all()) for x in others + [p, g])
    opt.bind([p], [g])
    opt.step()
    assert torch.allclose(p, torch.full_like(p, 7.0 - 0.125), rtol=0, atol=1e-5)


def test_what_waits_is_refused_under_capture(snk):
    """Step counts, reset and the choice of a model's optimizer; the capture goes on, with nothing of them in it."""
    p, g = torch.ones(300, device="cuda"), torch.ones(300, device="cuda")
    opt = snk.AdamW([p], [g], max_grad_norm=1.0)
    opt.step()
    assert opt.steps == 1
    model = snk.DQNModel(12, 3, n_frames=2, seed=3)
    held = model.use_adamw(lr=1e-3)
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.graph(graph, stream=side):
        for use in (lambda: opt.steps, lambda: setattr(opt, "steps", 7), opt.reset):
            with pytest.raises(snk.SnakeHipError, match="captured"):
                use()
        snk._lib.call("snk_set_stream", side.cuda_stream)
        try:
            for use in (model.use_rmsprop, model.use_adamw, lambda: held.steps, held.reset):
                with pytest.raises(snk.SnakeHipError, match="captured"):
                    use()
        finally:
            snk._lib.call("snk_set_stream", None)
        opt.step()
    moments = opt.state()["m"].numpy()
    assert opt.steps == 1 and moments.any()
    for t in (2, 3):
        graph.replay()
        torch.cuda.synchronize()
        assert opt.steps == t and np.all(np.abs(opt.state()["m"].numpy()[:300]) > np.abs(moments[:300]))
    assert held.steps == 0 and model.adamw is held
    model.use_rmsprop()


def test_autograd_sees_the_step(snk):
    """A graph that saved a parameter before the step refuses its backward pass, as after torch's own."""
    flat = torch.randn(2000, device="cuda")
    leaf = torch.nn.Parameter(torch.randn(500, device="cuda"))
    work = torch.zeros(500, dtype=torch.bfloat16, device="cuda")
    a, b = flat[:700], flat[1000:]
    g = [torch.randn(x.numel(), device="cuda") for x in (leaf, a, b)]
    opt = snk.AdamW([leaf, a, b], g)
    for how in (lambda: opt.step(), lambda: opt.step(g)):
        x = torch.randn(500, device="cuda", requires_grad=True)
        before = [t._version for t in (leaf, a, b, flat)]
        loss, whole = (x * leaf).sum(), (x * flat[:500]).sum()
        how()
        assert all(t._version > v for t, v in zip((leaf, a, b, flat), before))
        for y in (loss, whole):
            with pytest.raises(RuntimeError, match="inplace"):
                y.backward()
        (x * leaf).sum().backward()       # a graph of after the step is fine
    copied = snk.AdamW([torch.nn.Parameter(torch.randn(500, device="cuda"))], [g[0]], copies=[work])
    v = work._version
    copied.step()
    assert work._version > v
    out = torch.empty(opt.total, device="cuda")
    v = out._version
    opt.moments(None, out)
    assert out._version > v
    with torch.inference_mode():          # tensors that count nothing
        snk.AdamW([torch.ones(9, device="cuda")], [torch.ones(9, device="cuda")]).step()


def test_moments_into_overlapping_arrays_are_refused(snk):
    p, g = torch.ones(300, device="cuda"), torch.ones(300, device="cuda")
    opt = snk.AdamW([p], [g])
    x = torch.full((2 * opt.total,), 7.0, device="cuda")
    for a, b in ((0, 1), (opt.total - 1, 0), (5, 5)):
        with pytest.raises(snk.SnakeHipError, match="overlap"):
            opt.moments(x[a:a + opt.total], x[b:b + opt.total])
    for m, v in ((x.data_ptr() + 2, None), (None, x.data_ptr() + 1)):
        with pytest.raises(snk.SnakeHipError, match="aligned"):
            snk._lib.call("snk_adamw_moments", opt.handle, 0, m, v)
    assert bool((x == 7.0).all())
    opt.moments(x[opt.total:], x[:opt.total])
    assert not bool(x.any())


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("max_norm", [0.0, 1.0])
def test_nothing_to_step(snk, bits, max_norm):
    """Tensors without elements: steps are counted, the state is empty."""
    p, g = ([torch.empty(0, device="cuda"), torch.empty(3, 0, device="cuda")] for _ in range(2))
    opt = snk.AdamW(p, g, state_bits=bits, max_grad_norm=max_norm)
    opt.step()
    opt.step([x.bfloat16() for x in g])
    assert opt.steps == 2 and opt.total == 0 and opt.starts == [0, 0]
    assert all(x.numpy().size == (k == "norm") for k, x in opt.state().items())
    assert torch.as_tensor(opt.state()["m"], device="cuda").numel() == 0
    opt.moments(torch.empty(0, device="cuda"))
    opt.reset()
    assert opt.steps == 0


def test_a_loop_over_a_module(snk):
    """As a training loop uses it: autograd's own gradients, new ones every iteration, of parameters of any
    shape, on a side stream; the updates are the formula's, whatever the gradients' places."""
    gen = torch.Generator(device="cuda").manual_seed(9)
    net = torch.nn.Sequential(torch.nn.Linear(40, 33), torch.nn.Tanh(), torch.nn.Linear(33, 7)).cuda()
    params = list(net.parameters())
    sizes = [p.numel() for p in params]
    opt = snk.AdamW(params, lr=1e-2, weight_decay=[0.1 if p.dim() > 1 else 0.0 for p in params], max_grad_norm=0.5)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    kept = []
    with torch.cuda.stream(side):
        for t in range(1, 5):
            for p in params:
                p.grad = None
            x = torch.randn(16, 40, device="cuda", generator=gen)
            (net(x) ** 2).sum().backward()
            grads = [p.grad for p in params]
            kept.append(torch.empty(sizes[0], device="cuda"))   # takes the place of a gradient that was freed
            check_step(opt, [p.detach() for p in params], grads, sizes, [0.1, 0.0, 0.1, 0.0], t, lambda: opt.step(grads),
                       ptype="f32", lr=1e-2, b1=0.9, b2=0.999, eps=1e-8, max_norm=0.5)
            del grads
        side.synchronize()
    torch.cuda.current_stream().wait_stream(side)


def test_bound_gradients_are_not_unbound(snk):
    """A captured step would read at no address."""
    p, g = torch.ones(300, device="cuda"), torch.ones(300, device="cuda")
    opt = snk.AdamW([p], [g])
    where = (C.c_void_p * 1)(p.data_ptr())
    with pytest.raises(snk.SnakeHipError, match="are bound"):
        snk._lib.call("snk_adamw_bind", opt.handle, where, None, None)
    opt.step()
    assert opt.steps == 1 and bool((p < 1).all())
    own = snk.AdamW([g])
    snk._lib.call("snk_adamw_bind", own.handle, (C.c_void_p * 1)(g.data_ptr()), None, None)
    with pytest.raises(snk.SnakeHipError, match="no gradients"):
        snk._lib.call("snk_adamw_step", own.handle, 0.1, 1.0)
