"""The sampler on the GPU against its definition in 64 bits: equal indices, probabilities to fp32.

A reference answer whose margin (how near u or a filter's limit is to a step of the sums, relative
to the mass) is under 1e-9 may fall to either side and is left out; with random inputs that is rare,
and each test asserts how rare. The probability is a quotient of 64-bit sums whose entries are
rounded to 2^-(61 - log2 n) of the largest weight, rounded to fp32: half a step 2^-24, and 1e-9; where
the limit of top-p is that near to a step, S may or may not hold the entries within 1e-9 of it on
either side, 2e-9 more.
"""
import numpy as np
import pytest

import devrng
import sample_ref

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
TT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SETTINGS = [dict(), dict(temperature=0.3), dict(top_k=1), dict(top_k=5), dict(top_k=50, top_p=0.8), dict(top_p=0.9),
            dict(top_p=0.0), dict(min_p=0.1), dict(min_p=1.0), dict(top_k=700, top_p=0.95, min_p=0.01, temperature=1.7),
            dict(top_p=0.999, temperature=3.0), dict(temperature=0.0)]


def check(snk, x, u, mask=None, most_left_out=0, **how):
    """x [rows, n] torch tensor, how: numbers or arrays of one value per row."""
    rows, n = x.shape
    out = torch.full((rows + 2,), -7, dtype=torch.int32, device="cuda")
    prob = torch.full((rows + 2,), -7.0, device="cuda")
    dev = {k: torch.as_tensor(v, device="cuda") if isinstance(v, np.ndarray) else v for k, v in how.items()}
    got = snk.sample_logits(x, u, mask=mask, out=out[1:-1], prob=prob[1:-1], **dev)
    assert got.data_ptr() == out[1:-1].data_ptr()
    idx, pr = out.cpu().numpy(), prob.double().cpu().numpy()
    assert idx[0] == idx[-1] == -7 and pr[0] == pr[-1] == -7
    xs, us = x.double().cpu().numpy(), u.cpu().numpy()
    ms = None if mask is None else np.broadcast_to(mask.cpu().numpy(), xs.shape)
    left_out = 0
    for r in range(rows):
        one = {k: v[r] if isinstance(v, np.ndarray) else v for k, v in how.items()}
        i, p, margin = sample_ref.row(xs[r], us[r], mask=None if ms is None else ms[r], **one)
        if margin < 1e-9:
            left_out += 1
            continue
        assert idx[1 + r] == i, (r, idx[1 + r], i, margin, one)
        assert np.isnan(p) == np.isnan(pr[1 + r])
        if not np.isnan(p):
            assert abs(pr[1 + r] - p) <= (2.0 ** -24 + 3e-9) * p, (r, pr[1 + r], p)
    assert left_out <= most_left_out, left_out
    return idx[1:-1]


def logits(rows, n, dtype, seed, std=2.0, stride=None, offset=0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    stride = stride or n
    buf = torch.full((rows * stride + offset,), float("nan"), dtype=TT[dtype], device="cuda")   # never to be read
    x = buf[offset:offset + rows * stride].view(rows, stride)[:, :n]
    x.copy_(torch.randn(rows, n, device="cuda", generator=gen) * std)
    return x, torch.rand(rows, device="cuda", generator=gen)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("n", [1, 2, 3, 4, 5, 8, 9, 31, 63, 64, 65, 200, 511, 512, 513, 1000, 1024, 2047, 4097, 8193, 16385, 50021])
def test_sizes_and_settings(snk, dtype, n):
    for k, how in enumerate(SETTINGS):
        x, u = logits(6, n, dtype, 100 * n + k)
        # a quarter of 2^-9 steps of bf16 values may tie; the margin of distinct sums is about 1 / n / S
        check(snk, x, u, most_left_out=1, **how)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("n,stride,offset", [(7, 9, 1), (100, 101, 1), (700, 703, 3), (5000, 5001, 1), (33000, 33005, 2)])
def test_strides_and_alignment(snk, dtype, n, stride, offset):
    """Rows that start at any element; what lies between them is NaN and must not matter."""
    for how in (dict(), dict(top_k=20), dict(top_p=0.7), dict(min_p=0.05)):
        x, u = logits(9, n, dtype, n, stride=stride, offset=offset)
        gen = torch.Generator(device="cuda").manual_seed(n)
        mask = (torch.rand(9, stride, device="cuda", generator=gen) < 0.3)[:, :n]
        check(snk, x, u, most_left_out=1, **how)
        check(snk, x, u, mask=mask.to(torch.uint8) if n % 2 else mask, most_left_out=1, **how)
        check(snk, x, u, mask=mask[3].contiguous(), most_left_out=1, **how)


def test_one_row_for_all(snk):
    """An expanded row (stride 0), a thousand draws: the drawn shares are those of the weights, since
    the given u are a grid: an entry of probability p is hit by p 1000 +- 1 of them."""
    x, _ = logits(1, 300, "f32", 3, std=1.0)
    u = (torch.arange(1000, device="cuda") + 0.5) / 1000
    idx = check(snk, x.expand(1000, 300), u)
    p = torch.softmax(x[0].double(), 0).cpu().numpy()
    assert np.all(np.abs(np.bincount(idx, minlength=300) - 1000 * p) <= 1 + 1e-6)
    one = snk.sample_logits(x[0], u[:1])
    assert int(one[0]) == idx[0]


@pytest.mark.parametrize("n", [3, 8, 40, 600, 9000])
def test_rows_with_nothing_and_odd_values(snk, n):
    x, u = logits(24, n, "f32", n)
    mask = torch.zeros(24, n, dtype=torch.uint8, device="cuda")
    low, inf, nan = torch.finfo(torch.float32).min, float("inf"), float("nan")
    mask[0] = 1                                # nothing left
    x[1] = -inf                                # nothing left
    x[2, :], mask[2, :] = nan, 255             # NaN, all masked
    x[3, 0], mask[3, 0] = nan, 1               # NaN and infinity in masked places
    x[4, 0], mask[4, 0] = inf, 1
    x[5, n // 2] = nan                         # NaN in an allowed place
    x[6, n - 1] = inf                          # one infinite entry
    x[7, 0] = x[7, n - 1] = inf                # two
    x[8] = low                                 # the type's lowest everywhere
    x[9, 1:] = low                             # ... but for one
    x[10] = 0.25                               # all equal
    x[11, ::2], x[11, 1::2] = 0.0, -0.0        # equal zeros
    mask[12, : n - 1] = 1                      # only the last allowed
    x[13] = torch.arange(n, device="cuda") * 1e-42    # subnormal
    x[14] = -inf
    x[14, n // 2] = -1e30                      # one entry, far down
    x[15] = torch.where(torch.arange(n, device="cuda") % 3 == 0, 5.0, 1.0)
    u[16], u[17], u[18], u[19], u[20] = 0.0, 0.99999994, 1.0, nan, -3.0
    x[21] = 3e38
    x[22, 0], x[22, 1] = -nan, 1.0             # a NaN of the other sign
    x[23, 0], x[23, 1:] = -3e38, 3e38
    for how in (dict(), dict(top_k=2), dict(top_p=0.6), dict(min_p=0.5), dict(temperature=0.0), dict(temperature=1e-30),
                dict(temperature=1e30), dict(top_k=3, top_p=0.99, min_p=0.001)):
        check(snk, x, u, mask=mask, most_left_out=24, **how)   # equal entries put limits on exact steps
    idx = check(snk, x, u, mask=mask, top_p=0.6, most_left_out=24)
    assert idx[0] == idx[1] == idx[2] == idx[5] == idx[22] == -1 and idx[12] == n - 1 and idx[14] == n // 2 and idx[6] == n - 1
    assert min(idx[3], idx[4]) >= 1
    assert idx[7] in (0, n - 1)


@pytest.mark.parametrize("n", [6, 300, 3000, 70001])
def test_settings_of_each_row(snk, n):
    rng = np.random.default_rng(n)
    rows = 40
    x, u = logits(rows, n, "f16", n)
    how = dict(temperature=rng.uniform(0.2, 2, rows).astype(np.float32), top_k=rng.integers(0, 60, rows).astype(np.int32),
               top_p=rng.uniform(0.2, 1, rows).astype(np.float32), min_p=rng.uniform(0, 0.2, rows).astype(np.float32))
    how["top_k"][:4] = [-3, n, n + 9, 2 ** 31 - 1]          # off
    how["temperature"][4:7] = [0.0, -1.0, np.nan]           # the largest
    how["top_p"][7:11] = [1.0, 7.0, np.nan, -1.0]
    how["min_p"][11:14] = [-1.0, np.nan, 9.0]
    check(snk, x, u, most_left_out=4, **how)
    for key in how:
        check(snk, x, u, most_left_out=4, **{key: how[key]})


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("how", [dict(), dict(top_p=0.97), dict(top_k=1500), dict(top_k=64), dict(min_p=1e-4),
                                 dict(top_k=100000, top_p=0.999)])
def test_long_rows(snk, dtype, how):
    for rows, n in ((3, 262144), (2, 1_000_003)):
        x, u = logits(rows, n, dtype, n, std=1.5)
        check(snk, x, u, most_left_out=1, **how)


@pytest.mark.parametrize("n", [9, 100, 513, 2048, 2049, 5000, 9000])
def test_many_rows(snk, n):
    """Hundreds of rows take smaller workgroups (and thousands, for top-p, several launches): the same
    answers as the rows get in small calls, and the reference's on some."""
    rows = 3001 if n == 9000 else 600
    x, u = logits(rows, n, "f32", n)
    mask = torch.rand(n, device="cuda", generator=torch.Generator(device="cuda").manual_seed(n)) < 0.2
    for how in (dict(), dict(top_k=40), dict(top_p=0.9), dict(top_k=30, top_p=0.9, min_p=0.01), dict(min_p=0.02), dict(temperature=0.0)):
        got = snk.sample_logits(x, u, mask=mask, **how)
        for part in (slice(0, 20), slice(rows - 20, rows)):
            assert torch.equal(got[part], snk.sample_logits(x[part], u[part], mask=mask, **how)), how
            check(snk, x[part], u[part], mask=mask, most_left_out=1, **how)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("std", [0.0, 1e-3, 0.05, 0.5, 8.0])
def test_nucleus_of_any_shape(snk, dtype, std):
    """From all entries equal to a handful that hold everything; limits near both ends."""
    for n in (3000, 20000, 131072):
        x, u = logits(4, n, dtype, n, std=std)
        for p in (1e-6, 0.3, 0.9, 0.999, 0.9999999):
            # equal weights put the sums of the limit on whole numbers
            check(snk, x, u, most_left_out=4 if std == 0 else 1, top_p=p)
        check(snk, x, u, most_left_out=4 if std == 0 else 1, top_p=0.8, min_p=0.4, temperature=0.7)


def test_the_longest_row(snk):
    n = 2 ** 24
    x, u = logits(1, n, "bf16", 1, std=1.0)
    for how in (dict(top_k=30), dict(top_p=0.5), dict(min_p=0.3)):
        check(snk, x, u, most_left_out=1, **how)
    with pytest.raises(snk.SnakeHipError, match="logits a row"):
        snk.sample_logits(torch.zeros(n + 1, device="cuda"), torch.zeros(1, device="cuda"))


def test_many_ties(snk):
    """Few distinct values: cuts fall inside runs of equal entries, the lower indices stay."""
    gen = torch.Generator(device="cuda").manual_seed(8)
    for n in (8, 100, 511, 5000, 40000):
        x = torch.randint(0, 4, (16, n), device="cuda", generator=gen).float() * 0.7
        u = torch.rand(16, device="cuda", generator=gen)
        for how in (dict(top_k=n // 3 + 1), dict(top_p=0.61803), dict(top_k=n // 2 + 1, top_p=0.7717), dict(min_p=0.2)):
            check(snk, x, u, most_left_out=1, **how)


def test_offsets_past_32_bits(snk):
    """Rows whose elements lie past 2^32 bytes and past 2^31 elements."""
    n = 2 ** 20 + 1
    rows = 2100
    x = torch.empty(rows, n, dtype=torch.bfloat16, device="cuda").normal_(0, 2)
    u = torch.rand(rows, device="cuda")
    for how in (dict(top_k=20), dict()):
        got = snk.sample_logits(x, u, **how)
        part = slice(rows - 2, rows)
        check(snk, x[part], u[part], most_left_out=1, **how)
        assert torch.equal(got[part], snk.sample_logits(x[part], u[part], **how))


@pytest.mark.parametrize("rows,n", [(5, 3), (3, 400), (2, 30000), (70, 9000), (300, 2000)])
def test_captured_and_on_another_stream(snk, rows, n):
    """Replays of two captured calls and eager calls between them agree with eager calls."""
    how = dict(top_k=9, top_p=0.9)
    x, u = logits(rows, n, "f32", rows)
    y, v = logits(rows, n, "f32", rows + 1)
    fresh = [logits(rows, n, "f32", 50 + i) for i in range(4)]
    graphs = []
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    for a, b in ((x, u), (y, v)):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            out = snk.sample_logits(a, b, **how)
        graphs.append((g, out))
    for (fx, fu) in fresh:
        x.copy_(fx), u.copy_(fu), y.copy_(fx * 0.5), v.copy_(fu)
        for g, _ in graphs:
            g.replay()
        eager = snk.sample_logits(fx, fu, **how), snk.sample_logits(fx * 0.5, fu, **how)
        torch.cuda.synchronize()
        assert torch.equal(graphs[0][1], eager[0]) and torch.equal(graphs[1][1], eager[1])
    with torch.cuda.stream(side):
        torch.cuda._sleep(5_000_000)
        x.copy_(fresh[0][0]), u.copy_(fresh[0][1])
        late = snk.sample_logits(x, u, **how)
    side.synchronize()
    assert torch.equal(late, snk.sample_logits(fresh[0][0], fresh[0][1], **how))


@pytest.mark.parametrize("n", [3, 500, 20000])
def test_device_arrays(snk, n):
    x, u = logits(4, n, "f32", n)
    a, b = snk.DeviceArray.from_host(x.cpu().numpy()), snk.DeviceArray.from_host(u.cpu().numpy())
    assert np.array_equal(snk.sample_logits(a, b, top_k=7).numpy(), snk.sample_logits(x, u, top_k=7).cpu().numpy())


def test_python_refusals(snk):
    x, u = logits(4, 100, "f32", 0)
    for bad in (dict(logits=x.t(), u=u), dict(logits=x, u=u[:3]), dict(logits=x, u=u.double()), dict(logits=x.int(), u=u),
                dict(logits=x[None], u=u), dict(logits=x, u=u, mask=x), dict(logits=x, u=u, mask=x[:, :9] > 0),
                dict(logits=x, u=u, out=torch.zeros(4, device="cuda")), dict(logits=x, u=u, prob=u[:2]),
                dict(logits=x, u=u, temperature=u[:2]), dict(logits=x, u=u, top_k=u)):
        with pytest.raises(ValueError):
            snk.sample_logits(**bad)
    with pytest.raises(snk.SnakeHipError):
        snk.sample_logits(x, u, top_p=1.01)
    with pytest.raises(ValueError, match="mix"):
        snk.sample_logits(x, snk.DeviceArray(4, np.float32))


# ------------------------------------------------------------------ the policy over an env batch

@pytest.mark.parametrize("deep", [False, True])
def test_softmax_actions(snk, deep):
    n, seed = 300, 77
    game = snk.SnakeGame(12, 2, n_envs=n, autoreset=True)
    model = snk.DQNModel(12, 3, n_frames=2, seed=4, deep=deep)
    act = snk.DeviceArray(n, np.uint8)
    for t in range(3):
        q = model.q_env(game)
        for how in (dict(temperature=0.05), dict(temperature=0.0), dict(temperature=0.1, top_k=2), dict(top_p=0.5)):
            got = snk.softmax_actions(game, model, seed=seed, act=act, **how)
            for e in range(n):
                u = devrng.rng_uniform(devrng.rng_hash(seed, e, t))
                want, _, margin = sample_ref.row(q[e], u, **how)
                assert margin < 1e-9 or got[e] == want
        assert np.array_equal(snk.softmax_actions(game, model, temperature=0.0), snk.epsilon_greedy(game, model, 0.0))
        snk.step_indices_dev(game, act.ptr)


def test_an_iteration_of_both_ends(snk):
    """Acting by the softmax policy and learning by AdamW, together as a training loop uses them:
    every action against the definition, every update against the formula."""
    import adamw_ref
    n, seed = 128, 5
    game = snk.SnakeGame(12, 2, n_envs=n, autoreset=True)
    rb = snk.ReplayBuffer(2048, board_size=12, n_frames=2)
    model = snk.DQNModel(12, 3, n_frames=2, seed=8)
    opt = model.use_adamw(lr=1e-3, weight_decay=0.01, max_grad_norm=1.0)
    sizes = [288, 16, 4608, 32, 73728, 64, 49 * 4096, 64, 192, 3]
    perm, (starts, total) = model.flux_index(), adamw_ref.places(sizes)
    ends = np.cumsum([0] + sizes)

    def layout(flux):
        out = np.zeros(total)
        for at, a, b in zip(starts, ends, ends[1:]):
            out[at:at + b - a] = flux[perm][a:b]
        return out

    wd = layout(np.ones(model.P, np.float32)) * 0
    for i, (at, s) in enumerate(zip(starts, sizes)):
        wd[at:at + s] = 0.0 if i % 2 else 0.01
    act, updates = snk.DeviceArray(n, np.uint8), 0
    for t in range(6):
        q = model.q_env(game)
        got = snk.softmax_actions(game, model, temperature=0.2, top_k=2, seed=seed, act=act)
        for e in range(n):
            u = devrng.rng_uniform(devrng.rng_hash(seed, e, t))
            want, _, margin = sample_ref.row(q[e], u, temperature=0.2, top_k=2)
            assert margin < 1e-9 or got[e] == want
        snk.step_indices_dev(game, act.ptr, replay=rb)
        if t < 2:
            continue
        idx, B = snk.sample(rb, seed=t)
        st = {k: v.numpy() for k, v in opt.state().items()}
        p = layout(model.get_params())
        loss = model.update(rb, idx, B)
        updates += 1
        want = adamw_ref.Step(p, layout(model.grad), st["m"], st["v"], updates, lr=1e-3, b1=0.9, b2=0.999, eps=1e-8, wd=wd,
                              max_norm=1.0)
        assert np.all(np.abs(layout(model.get_params()) - want.p) <= want.ep) and np.isfinite(loss)
    assert opt.steps == updates


@pytest.mark.parametrize("n", [9, 2049])
def test_more_rows_than_one_grid(snk, n):
    """Rows past 2^22, which take a second launch, answer as a call of their own."""
    rows, last = (1 << 22) + 300, 400
    gen = torch.Generator(device="cuda").manual_seed(n)
    x = torch.randn(n, device="cuda", generator=gen).to(torch.float16)
    u = torch.rand(rows, device="cuda", generator=gen)
    prob, want_prob = torch.empty(rows, device="cuda"), torch.empty(last, device="cuda")
    got = snk.sample_logits(x.expand(rows, n), u, prob=prob)
    want = snk.sample_logits(x.expand(last, n), u[-last:].contiguous(), prob=want_prob)
    assert torch.equal(got[-last:], want) and torch.equal(prob[-last:], want_prob)
    want = snk.sample_logits(x.expand(last, n), u[:last].contiguous(), prob=want_prob)
    assert torch.equal(got[:last], want) and torch.equal(prob[:last], want_prob)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("n", [10, 16, 40, 128, 129, 256, 257, 1023, 1025, 2048, 2049, 3333, 4095, 4096])
def test_rows_in_registers(snk, dtype, n):
    """Few rows and many, of the sizes at which a row's share of waves changes; what is not the row's is NaN."""
    for k, how in enumerate(SETTINGS + [dict(top_k=33, top_p=0.6), dict(top_k=64, top_p=0.99, min_p=0.02), dict(top_k=9, temperature=9.0)]):
        x, u = logits(6, n, dtype, 7 * n + k, stride=n + 3, offset=1)
        check(snk, x, u, most_left_out=1, **how)
        x, u = logits(700, n, dtype, 9 * n + k)
        x[5] = -torch.inf
        x[6, : n // 2] = torch.inf
        x[7] = 0.25
        x[8, n // 3] = torch.nan
        x[9, n - 1] = -torch.inf
        x[10, 1:] = -torch.inf
        mask = torch.rand(700, n, device="cuda", generator=torch.Generator(device="cuda").manual_seed(n)) < 0.3
        mask[11, : n // 2] = True
        got = snk.sample_logits(x, u, mask=mask, **how)
        rows = slice(0, 24)
        assert torch.equal(got[rows], snk.sample_logits(x[rows], u[rows], mask=mask[rows], **how)), how
        check(snk, x[rows], u[rows], mask=mask[rows], most_left_out=2, **how)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("n", [20, 64, 500, 900, 2000, 4000])
def test_ties_at_the_cut(snk, dtype, n):
    """Few distinct values of either sign: cuts that split a run of equal entries, in index order."""
    gen = torch.Generator(device="cuda").manual_seed(n)
    x = (torch.randint(-3, 4, (600, n), device="cuda", generator=gen) * 0.5).to(TT[dtype])
    u = torch.rand(600, device="cuda", generator=gen)
    for how in (dict(top_k=7), dict(top_k=n // 2), dict(top_p=0.4), dict(top_p=0.9, min_p=0.1), dict(top_k=60, top_p=0.7),
                dict(top_k=n // 2 + 1, top_p=0.5)):
        got = snk.sample_logits(x, u, **how)
        assert torch.equal(got[:20], snk.sample_logits(x[:20], u[:20], **how)), how
        check(snk, x[:20], u[:20], most_left_out=1, **how)


@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("n", [8192, 8193, 20011, 32767, 32768, 32769])
def test_rows_scanned_by_their_workgroup(snk, dtype, n):
    """Up to 32,768 entries, four pieces of 512 a wave, the row's end inside any of them; as many rows
    take the scan's own launch."""
    for k, how in enumerate(SETTINGS):
        x, u = logits(520, n, dtype, n + k, stride=n + 1, offset=1)
        x[3] = -torch.inf
        x[4, 1000:] = -torch.inf
        x[5, :-1] = -torch.inf
        mask = torch.rand(n, device="cuda", generator=torch.Generator(device="cuda").manual_seed(n)) < 0.3
        few = slice(0, 9)
        check(snk, x[few], u[few], mask=mask, most_left_out=1, **how)
        got = snk.sample_logits(x, u, mask=mask, **how)
        assert (got[few] != snk.sample_logits(x[few], u[few], mask=mask, **how)).sum() <= 1, how   # sums in another order


@pytest.mark.parametrize("n", [700, 1024, 4097, 9000, 40000])
def test_rows_by_the_card(snk, n):
    """The numbers of rows at which a row's workgroup shrinks give the same answers."""
    x, u = logits(1030, n, "bf16", n)
    mask = torch.rand(n, device="cuda", generator=torch.Generator(device="cuda").manual_seed(n)) < 0.1
    for how in (dict(), dict(top_k=40), dict(top_p=0.9), dict(top_k=30, top_p=0.9), dict(min_p=0.02), dict(top_k=90, min_p=0.1)):
        calls = [snk.sample_logits(x[:rows], u[:rows], mask=mask, **how)[:250] for rows in (250, 256, 257, 512, 513, 767, 768, 1030)]
        check(snk, x[:10], u[:10], mask=mask, most_left_out=1, **how)
        for got in calls[1:]:
            assert (got != calls[0]).sum() <= 1, how   # whole rows' masses are added in another order


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("n", [4097, 8192, 12345, 33000, 70001])
def test_large_top_k(snk, dtype, n):
    """Cuts that the maxima of 64 do not bound: by the maxima of 8, or by the whole row."""
    for rows in (5, 300, 600):
        x, u = logits(rows, n, dtype, n + rows)
        x[1] = -torch.inf
        x[2, 3000:] = -torch.inf
        x[3] = torch.round(x[3])                 # many ties
        x[4, ::2] = x[4, 0]
        mask = torch.rand(n, device="cuda", generator=torch.Generator(device="cuda").manual_seed(n)) < 0.2
        part = slice(0, 6)
        for how in (dict(top_k=n // 64 + 1), dict(top_k=n // 64 - 3, top_p=0.9), dict(top_k=700), dict(top_k=1000, top_p=0.7),
                    dict(top_k=1990, min_p=0.003), dict(top_k=2000, top_p=0.95, min_p=0.001), dict(top_k=4050), dict(top_k=n - 1)):
            got = snk.sample_logits(x, u, mask=mask, **how)
            assert torch.equal(got[part], snk.sample_logits(x[part], u[part], mask=mask, **how)), how
            check(snk, x[part], u[part], mask=mask, most_left_out=2, **how)


@pytest.mark.parametrize("n", [3, 40, 600, 3000, 4097, 20000, 70001])
def test_temperatures_at_the_ends(snk, n):
    """The least and the largest temperatures that fp32 holds, under every filter."""
    for t in (1e-45, 1e-38, 1e-20, 1e20, 3e38):
        for how in (dict(), dict(min_p=0.3), dict(min_p=1.0), dict(top_k=3, min_p=0.3), dict(top_p=0.5), dict(top_k=2, top_p=0.5)):
            for rows in (4, 300):
                x, u = logits(rows, n, "f32", n)
                got = snk.sample_logits(x, u, temperature=t, **how)
                assert int(got.min()) >= 0 and int(got.max()) < n, (t, how)
                if t < 1:
                    assert torch.equal(got.long(), x.argmax(1)), (t, how)
                else:
                    check(snk, x[:4], u[:4], temperature=t, most_left_out=4, **how)


def test_threads_at_once(snk):
    """Two operators on threads and streams of their own: each call keeps its thread's stream."""
    import threading
    x, u = logits(64, 3000, "bf16", 1)
    p0, g = torch.randn(50_001, device="cuda"), torch.randn(50_001, device="cuda")
    want_index, want_p = snk.sample_logits(x, u, top_k=20, top_p=0.9), p0.clone()
    same = snk.AdamW([want_p], [g], state_bits=8)
    for _ in range(20):
        same.step()
    torch.cuda.synchronize()
    errors = []

    def run(which):
        try:
            stream = torch.cuda.Stream()
            with torch.cuda.stream(stream):
                if which % 2:
                    for _ in range(50):
                        got = snk.sample_logits(x, u, top_k=20, top_p=0.9)
                    stream.synchronize()
                    assert torch.equal(got, want_index)
                else:
                    p = p0.clone()
                    opt = snk.AdamW([p], [g], state_bits=8)
                    for _ in range(20):
                        opt.step()
                    stream.synchronize()
                    assert torch.equal(p, want_p)
        except BaseException as e:   # noqa: BLE001 - reported by the test's own thread
            errors.append(e)

    threads = [threading.Thread(target=run, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors


@pytest.mark.parametrize("rows", [6, 300, 600])
@pytest.mark.parametrize("n", [7, 300, 3000, 5000, 20000, 70001])
def test_distances_past_fp32(snk, rows, n):
    """Logits 6e38 apart weigh e^-2 of each other at a temperature of 3e38: kept as any others are."""
    x, u = logits(rows, n, "f32", n)
    u[:6] = torch.tensor([0.0, 0.3, 0.6, 0.9, 0.99, 0.999], device="cuda")
    x[:] = -3e38
    x[:, 0] = 3e38
    x[1, n // 2] = 3e38
    x[2, : n // 2] = 1e38
    x[3, 1:4] = -torch.inf
    x[4] = torch.linspace(-3.4e38, 3.4e38, n, device="cuda")
    mask = torch.zeros(n, dtype=torch.bool, device="cuda")
    mask[n - 1] = True
    for t in (3e38, 1e38, np.float32(np.inf)):
        t = np.full(rows, t, np.float32) if np.isinf(t) else float(t)
        for how in (dict(top_k=5), dict(top_k=1500), dict(min_p=0.1), dict(min_p=1e-5), dict(top_p=0.9), dict(top_k=40, top_p=0.8),
                    dict()):
            # equal weights put the limits on whole numbers
            check(snk, x[:6], u[:6], mask=mask, most_left_out=6, temperature=t[:6] if isinstance(t, np.ndarray) else t, **how)
            dev = torch.as_tensor(t, device="cuda") if isinstance(t, np.ndarray) else t
            got = snk.sample_logits(x, u, mask=mask, temperature=dev, **how)
            few = snk.sample_logits(x[:6], u[:6], mask=mask, temperature=dev[:6] if isinstance(t, np.ndarray) else t, **how)
            assert (got[:6] != few).sum() <= 1, (t, how)   # whole rows' masses are added in another order
    got = snk.sample_logits(x[:6], u[:6], temperature=3e38, top_k=5)
    assert got[5] == 4   # of weights 1 and four e^-2, at 0.999


def test_autograd_sees_the_outputs(snk):
    """An embedding that saved the drawn indices refuses its backward pass after the next draw into them."""
    x, u = logits(4, 100, "f32", 0)
    out, prob = torch.zeros(4, dtype=torch.int32, device="cuda"), torch.zeros(4, device="cuda")
    table = torch.randn(100, 8, device="cuda", requires_grad=True)
    loss = torch.nn.functional.embedding(out, table).sum()
    versions = out._version, prob._version
    snk.sample_logits(x, u, out=out, prob=prob)
    assert out._version > versions[0] and prob._version > versions[1]
    with pytest.raises(RuntimeError, match="inplace"):
        loss.backward()


def test_softmax_actions_with_settings_of_each_env(snk):
    n, seed = 200, 31
    rng = np.random.default_rng(2)
    game = snk.SnakeGame(12, 2, n_envs=n, autoreset=True)
    model = snk.DQNModel(12, 3, n_frames=2, seed=4)
    how = dict(temperature=rng.uniform(0.0, 0.2, n).astype(np.float32), top_k=rng.integers(0, 4, n).astype(np.int32),
               top_p=rng.uniform(0.3, 1, n).astype(np.float32), min_p=rng.uniform(0, 0.5, n).astype(np.float32))
    q = model.q_env(game)
    for keys in (list(how), ["temperature"], ["top_k", "min_p"]):
        dev = {k: snk.DeviceArray.from_host(how[k]) for k in keys}
        got = snk.softmax_actions(game, model, seed=seed, **dev)
        for e in range(n):
            u = devrng.rng_uniform(devrng.rng_hash(seed, e, 0))
            want, _, margin = sample_ref.row(q[e], u, **{k: how[k][e] for k in keys})
            assert margin < 1e-9 or got[e] == want
    model.set_params(np.full(model.P, np.nan, np.float32))
    assert not snk.softmax_actions(game, model, seed=seed).any()


@pytest.mark.parametrize("n", [5, 900, 3000, 70001, 1 << 22])
@pytest.mark.parametrize("units", [0.4, 0.6, 1.5, 2.45])
def test_stated_accuracy(snk, n, units):
    """One entry that holds nearly all and many of about a unit, where rounding to units shows most: sums,
    probabilities and answers are within the header's bounds. Each entry is off by half a unit and 4e-12 of
    itself, so S by n / 2 units and 4e-12 S; the probability's quotient by the two and fp32's half a step;
    the sum up to the answer, and u S, by S's error each."""
    s = min(51, 61 - int(np.ceil(np.log2(n))))
    x = torch.full((1, n), float(np.log(units) - s * np.log(2)), device="cuda")
    x[0, n // 3] = 0.0
    w = np.exp(x[0].double().cpu().numpy())
    upto = np.cumsum(w)          # in order: off by n 2^-53 S at most
    S = upto[-1]
    wild = n / 2 * 2.0 ** -s + (4e-12 + n * 2.0 ** -53) * S
    plain = n > 4096             # unrounded sums without a filter
    prob = torch.empty(1, device="cuda")
    for how in (dict(), dict(top_k=n - 1), dict(min_p=1e-30), dict(top_p=0.99999994)):
        # (entries that are never drawn count in unrounded sums: the answer is off by their mass there)
        error = (1e-11 + n * 2.0 ** -53) * S if plain and not how and units >= 0.5 else wild
        # of the small ones, top-p may drop those of the highest indices: a mass of 1 - p, one entry, and the
        # errors of its limit and of what stays
        low = S * (1 - float(np.float32(0.99999994))) + w[0] + 2 * error if "top_p" in how else 0.0
        for u in (0.0, 0.25, 0.5, 0.999, 0.99999, 0.99999994):
            uu = torch.tensor([u], device="cuda")
            i = int(snk.sample_logits(x, uu, prob=prob, **how)[0])
            t = float(uu[0]) * S
            if "top_k" in how:   # all but the last of the small ones
                t -= float(uu[0]) * w[-1]
            assert 0 <= i < n and w[i] >= 0.5 * 2.0 ** -s * (1 - 1e-9)
            assert upto[i] > t - low - 2 * error and upto[i] - w[i] <= t + low + 2 * error, (how, u, i)
            kept = S - (w[-1] if "top_k" in how else 0.0) - low
            p = float(prob[0])
            assert w[i] / (S + error) * (1 - 2.0 ** -24 - 4e-12) <= p <= w[i] / (kept - error) * (1 + 2.0 ** -24 + 4e-12), (how, u)
