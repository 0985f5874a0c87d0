"""The AdamW step and the sampler as measured operators.

Each case is one pass through one operator on data of a stated size. `run` computes it in plain
torch operations, or through the package where `own` is true. A case is a dict:

  op "adamw":  sizes (text, "count*size" or "size" joined by commas: the tensors' element counts),
               param / grad (element types), bits (32 or 8: the moments' storage), clip (the largest
               global gradient norm, 0 = no norm pass)
  op "sample": rows, n, dtype, temperature, top_k, top_p, min_p, mask (a byte per logit, about a tenth
               of them forbidden), each_row (the four settings differ from row to row), spread (the
               standard deviation of the logits)

The tensors of an AdamW case are views into one flat buffer, each on a multiple of 256 elements, as
the packed parameter vector of a model is.
"""
import itertools
import math

import torch

own = False

PAD = 256                     # every tensor starts on a multiple of this many elements
LR, B1, B2, EPS, WD = 3e-4, 0.9, 0.999, 1e-8, 0.01
STEPS = 1000                  # optimizer steps taken before the measured one
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
BYTES = {"f32": 4, "bf16": 2, "f16": 2}

# the parameter tensors of this repository's two Q-nets (board side 12 and 20, two frames)
QNET = "288,16,4608,32,73728,64,200704,64,192,3"
DEEP = "576,32,9216,32,18432,64,147456,64,921600,64,192,3"
# eight transformer blocks of width 1024 (four square products, two of the feed-forward layer, two
# norms) and an embedding of 32,000 rows: 133 M parameters in 65 tensors
BLOCKS = "32768000,32*1048576,16*4194304,16*1024"


def listed():
    return [
        # one update of the 12 x 12 Q-net: ten tensors, 280 k parameters: a few microseconds of traffic
        dict(name="adamw qnet", op="adamw", sizes=QNET, param="f32", grad="f32", bits=32, clip=1.0),
        # the same net with no norm pass and 8-bit moments
        dict(name="adamw8 qnet", op="adamw", sizes=QNET, param="f32", grad="f32", bits=8, clip=0.0),
        # the deeper bf16-forward net keeps fp32 weights: 1.1 M parameters
        dict(name="adamw8 deep", op="adamw", sizes=DEEP, param="f32", grad="f32", bits=8, clip=1.0),
        # adapters and norms: many small tensors of odd sizes
        dict(name="adamw many small", op="adamw", sizes="100*777,100*4099,60*33,1*1", param="f32", grad="bf16", bits=32,
             clip=1.0),
        # pre-training steps of a 133 M parameter model, fp32 weights and bf16 gradients
        dict(name="adamw blocks", op="adamw", sizes=BLOCKS, param="f32", grad="bf16", bits=32, clip=1.0),
        # ... with bf16 weights and 8-bit moments
        dict(name="adamw8 blocks", op="adamw", sizes=BLOCKS, param="bf16", grad="bf16", bits=8, clip=1.0),
        # exploration over a lockstep batch of games: three Q-values each
        dict(name="sample actions", op="sample", rows=65536, n=3, dtype="f32", temperature=0.5, top_k=0, top_p=1.0,
             min_p=0.0, mask=False, each_row=False, spread=1.0),
        # one request, one token
        dict(name="sample one row", op="sample", rows=1, n=32000, dtype="bf16", temperature=0.8, top_k=50, top_p=0.95,
             min_p=0.0, mask=False, each_row=False, spread=2.0),
        # a few requests over a large vocabulary, nucleus only
        dict(name="sample nucleus", op="sample", rows=8, n=131072, dtype="f32", temperature=1.0, top_k=0, top_p=0.9,
             min_p=0.0, mask=False, each_row=False, spread=2.5),
        # a serving batch whose requests bring their own settings, under a grammar's mask
        dict(name="sample own settings", op="sample", rows=128, n=50021, dtype="f16", temperature=0.9, top_k=40,
             top_p=0.95, min_p=0.02, mask=True, each_row=True, spread=2.5),
        # a large batch, min-p
        dict(name="sample min-p", op="sample", rows=512, n=32003, dtype="bf16", temperature=1.2, top_k=0, top_p=1.0,
             min_p=0.05, mask=False, each_row=False, spread=2.5),
        # rollouts that draw from the whole distribution
        dict(name="sample whole", op="sample", rows=256, n=131072, dtype="bf16", temperature=1.0, top_k=0, top_p=1.0,
             min_p=0.0, mask=False, each_row=False, spread=2.0),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    if rng.random() < 0.5:
        left, groups = _log(rng, 2_000, 100_000_000), []
        for _ in range(rng.randint(1, 6)):
            count = _log(rng, 1, 40)
            size = max(1, min(_log(rng, 1, 8_000_000) | rng.randint(0, 1), left // count))
            groups.append("%d*%d" % (count, size))
            left -= count * size
            if left < 64:
                break
        return dict(op="adamw", sizes=",".join(groups), param=rng.choice(["f32", "f32", "bf16", "f16"]),
                    grad=rng.choice(["f32", "bf16"]), bits=rng.choice([32, 8]), clip=rng.choice([0.0, 1.0]))
    n = _log(rng, 2, 200_000)
    rows = _log(rng, 1, max(1, min(65536, 30_000_000 // n)))
    return dict(op="sample", rows=rows, n=n, dtype=rng.choice(["f32", "bf16", "f16"]),
                temperature=round(rng.uniform(0.3, 1.5), 2), top_k=rng.choice([0, 1, _log(rng, 2, 2000)]),
                top_p=rng.choice([1.0, round(rng.uniform(0.3, 0.99), 2)]),
                min_p=rng.choice([0.0, round(rng.uniform(0.001, 0.2), 3)]), mask=rng.random() < 0.3,
                each_row=rng.random() < 0.3, spread=round(rng.uniform(0.5, 3.0), 2))


# ------------------------------------------------------------------ inputs

def _sizes(case):
    out = []
    for part in case["sizes"].split(","):
        count, _, size = part.rpartition("*")
        out += [int(size)] * (int(count) if count else 1)
    return out


def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _prepare_adamw(case, seed):
    gen = _generator(seed)
    sizes = _sizes(case)
    padded = [-(-s // PAD) * PAD for s in sizes]
    starts = [0, *itertools.accumulate(padded)]
    total = starts.pop()
    used = torch.zeros(total, dtype=torch.bool, device="cuda")
    decay = torch.zeros(total, dtype=torch.float32, device="cuda")
    wds = [WD if s >= 256 else 0.0 for s in sizes]           # biases and norms are not decayed
    for at, s, wd in zip(starts, sizes, wds):
        used[at:at + s] = True
        decay[at:at + s] = wd

    def normal(std):
        return torch.randn(total, device="cuda", generator=gen) * std * used

    p = normal(0.05).to(DTYPES[case["param"]])
    # gradients with a heavy tail, and an element in five that has none
    g = normal(1e-3) * torch.rand(total, device="cuda", generator=gen).clamp_min(0.05).rsqrt()
    g = (g * (torch.rand(total, device="cuda", generator=gen) > 0.2)).to(DTYPES[case["grad"]])
    m, v = normal(3e-4), normal(1e-3).square()
    state = dict(case=case, p=p, g=g, used=used, decay=decay, t=STEPS, seed=seed & 0xFFFF)
    if case["bits"] == 8:
        mb, vb = m.view(-1, PAD), v.view(-1, PAD)
        ms, vs = mb.abs().amax(1), vb.amax(1)
        a = (mb.abs() / ms.clamp_min(1e-30)[:, None]).sqrt().mul(127).round() * mb.sign()
        b = (vb / vs.clamp_min(1e-30)[:, None]).sqrt().sqrt().mul(255).round()
        b = torch.maximum(b, (vb > 0).to(b.dtype))
        state |= dict(m=a.to(torch.int8).view(-1), v=b.to(torch.uint8).view(-1), ms=ms, vs=vs)
    else:
        state |= dict(m=m, v=v)
    if own:
        import snake_amd
        params = [p[at:at + s] for at, s in zip(starts, sizes)]
        opt = snake_amd.AdamW(params, lr=LR, betas=(B1, B2), eps=EPS, weight_decay=wds, state_bits=case["bits"],
                              max_grad_norm=case["clip"], seed=state["seed"])
        view = {k: torch.as_tensor(x, device="cuda") for k, x in opt.state().items()}
        for name, key in (("m", "m"), ("v", "v"), ("m_scale", "ms"), ("v_scale", "vs")):
            if name in view:
                view[name].copy_(state[key])
        opt.steps = STEPS
        state |= dict(opt=opt, view=view, grads=[g[at:at + s] for at, s in zip(starts, sizes)])
        if case["bits"] == 8:
            state["values"] = [torch.empty(total, dtype=torch.bfloat16, device="cuda") for _ in range(2)]
    return state


def _prepare_sample(case, seed):
    gen = _generator(seed)
    rows, n = case["rows"], case["n"]
    x = torch.randn(rows, n, device="cuda", generator=gen) * case["spread"]
    if n > 64:   # a handful of words stand out, as after a prompt
        at = torch.randint(0, n, (rows, 16), device="cuda", generator=gen)
        x.scatter_add_(1, at, torch.rand(rows, 16, device="cuda", generator=gen) * 4 * case["spread"])
    state = dict(case=case, x=x.to(DTYPES[case["dtype"]]), u=torch.rand(rows, device="cuda", generator=gen), mask=None)
    if case["mask"]:
        mask = torch.rand(rows, n, device="cuda", generator=gen) < 0.1
        mask[:, 0] = False
        if rows > 1:
            mask[rows // 2] = True    # a row with nothing left
        state["mask"] = mask.to(torch.uint8)
    for key in ("temperature", "top_p", "min_p"):
        state[key] = torch.full((rows,), case[key], device="cuda")
    state["top_k"] = torch.full((rows,), case["top_k"], dtype=torch.int32, device="cuda")
    if case["each_row"]:
        turn = torch.rand(4, rows, device="cuda", generator=gen)
        state |= dict(temperature=state["temperature"] * (0.5 + 0.5 * turn[0]),
                      top_k=(state["top_k"] * (0.5 + 0.5 * turn[1])).ceil().to(torch.int32),
                      top_p=1 - (1 - state["top_p"]) * turn[2], min_p=state["min_p"] * turn[3])
    if own:
        import snake_amd
        state["sample"] = snake_amd.sample_logits
        state["out"] = torch.empty(rows, dtype=torch.int32, device="cuda")
        state["prob"] = torch.empty(rows, dtype=torch.float32, device="cuda")
    return state


def prepare(case, seed):
    return _prepare_adamw(case, seed) if case["op"] == "adamw" else _prepare_sample(case, seed)


# ------------------------------------------------------------------ the plain forms

def _shr(x, k):
    return (x >> k) & ((1 << (64 - k)) - 1)


def _i64(x):
    return x - (1 << 64) if x >= 1 << 63 else x


def _mix(x):
    """splitmix64 on int64 tensors (products wrap)."""
    z = x + _i64(0x9E3779B97F4A7C15)
    z = (z ^ _shr(z, 30)) * _i64(0xBF58476D1CE4E5B9)
    z = (z ^ _shr(z, 27)) * _i64(0x94D049BB133111EB)
    return z ^ _shr(z, 31)


def _bits16(seed, t, total):
    """The 16 random bits of every element's rounding: four to a hash of (seed, step, index / 4)."""
    key = _mix(torch.full((1,), _i64((seed ^ (t * 0xD1B54A32D192ED03)) & ((1 << 64) - 1)), dtype=torch.int64,
                          device="cuda"))
    h = _mix(key ^ torch.arange(total // 4, dtype=torch.int64, device="cuda"))
    return torch.stack([_shr(h, 16 * j) & 0xFFFF if j else h & 0xFFFF for j in range(4)], 1).view(-1)


def _plain_adamw(s):
    case = s["case"]
    s["t"] += 1
    t = s["t"]
    g = s["g"].float()
    out = {}
    if case["clip"]:
        norm = g.double().square().sum().sqrt()
        g = g * torch.clamp(case["clip"] / norm, max=1.0).float()
        out["norm"] = norm.float().view(1)
    if case["bits"] == 8:
        a, b = s["m"].view(-1, PAD).float(), s["v"].view(-1, PAD).float()
        m = (a * a.abs() / 16129 * s["ms"][:, None]).view(-1)
        v = ((b / 255).square().square() * s["vs"][:, None]).view(-1)
    else:
        m, v = s["m"], s["v"]
    m = m * B1 + g * (1 - B1)
    v = v * B2 + g * g * (1 - B2)
    p = s["p"].float()
    step = (m / (1 - B1 ** t)) / ((v / (1 - B2 ** t)).sqrt() + EPS)
    s["p"].copy_(p - LR * (step + s["decay"] * p))
    if case["bits"] == 8:
        mb, vb = m.view(-1, PAD), v.view(-1, PAD)
        ms, vs = mb.abs().amax(1, keepdim=True), vb.amax(1, keepdim=True)
        a = (mb.abs() / ms.clamp_min(1e-38)).sqrt().mul(127).round() * mb.sign()
        ratio = vb / vs.clamp_min(1e-38)
        low = (ratio.sqrt().sqrt() * 255).floor().clamp_max(254)
        lo, hi = (low / 255).square().square(), ((low + 1) / 255).square().square()
        up = _bits16(s["seed"], t, m.numel()).view(-1, PAD) < (ratio - lo) / (hi - lo) * 65536
        b = torch.maximum(low + up, (vb > 0).float())
        s["m"], s["v"] = a.to(torch.int8).view(-1), b.to(torch.uint8).view(-1)
        s["ms"], s["vs"] = ms.view(-1), vs.view(-1)
        out |= dict(m_scale=s["ms"], v_scale=s["vs"], m=(a * a.abs() / 16129 * ms).bfloat16().view(-1),
                    v=((b / 255).square().square() * vs).bfloat16().view(-1))
    else:
        s["m"], s["v"] = m, v
        out |= dict(m=m, v=v)
    return out | dict(p=s["p"])


def _plain_sample(s):
    x = s["x"].float()
    if s["mask"] is not None:
        x = x.masked_fill(s["mask"] != 0, -torch.inf)
    rows, n = x.shape
    order = torch.sort(x, dim=1, descending=True, stable=True)     # equal logits: the lower index first
    z = order.values.double() / s["temperature"].double()[:, None]
    w = (z - z[:, :1]).exp().nan_to_num(0.0)                       # a row with nothing left: all zero
    rank = torch.arange(n, device="cuda")
    k = torch.where(s["top_k"] > 0, s["top_k"], n).long()
    w = w * (rank < k[:, None])
    before = w.cumsum(1) - w
    keep = (before < s["top_p"].double()[:, None] * w.sum(1, keepdim=True)) | (s["top_p"][:, None] >= 1)
    w = w * (keep & (w >= s["min_p"].double()[:, None]))
    w = torch.zeros_like(w).scatter_(1, order.indices, w)          # back in the order of the indices
    up_to = w.cumsum(1)
    whole = up_to[:, -1:]
    index = (up_to <= s["u"].double()[:, None] * whole).sum(1, keepdim=True).clamp_max(n - 1)
    prob = w.gather(1, index) / whole
    none = whole == 0
    return dict(index=torch.where(none, -1, index).int().view(-1), prob=torch.where(none, 0.0, prob).float().view(-1))


def run(state):
    case = state["case"]
    if case["op"] == "adamw":
        if not own:
            return _plain_adamw(state)
        opt = state["opt"]
        opt.step(state["grads"])
        out = dict(p=state["p"], m=state["view"]["m"], v=state["view"]["v"])
        if case["bits"] == 8:
            opt.moments(*state["values"])
            out |= dict(m=state["values"][0], v=state["values"][1], m_scale=state["view"]["m_scale"],
                        v_scale=state["view"]["v_scale"])
        if case["clip"]:
            out["norm"] = state["view"]["norm"]
        return out
    if not own:
        return _plain_sample(state)
    if case["each_row"]:
        how = {k: state[k] for k in ("temperature", "top_k", "top_p", "min_p")}
    else:
        how = {k: case[k] for k in ("temperature", "top_k", "top_p", "min_p")}
    state["sample"](state["x"], state["u"], mask=state["mask"], out=state["out"], prob=state["prob"], **how)
    return dict(index=state["out"], prob=state["prob"])


def work(case):
    if case["op"] == "adamw":
        n = sum(_sizes(case))
        per = 2 * BYTES[case["param"]] + BYTES[case["grad"]]
        # 8-bit moments are read and written, and their values returned in bf16; the scales are 16 B a block
        per += 16 if case["bits"] == 32 else 4 + 4 + 16 / PAD
        return {"bytes": n * per, "flops": n * (20 if case["bits"] == 32 else 50)}
    n = case["rows"] * case["n"]
    return {"bytes": n * (BYTES[case["dtype"]] + (1 if case["mask"] else 0)) + case["rows"] * 12, "flops": n * 4}


# ------------------------------------------------------------------ the definitions in 64 bits

def _exact_adamw(case, seed):
    s = _prepare_adamw(case, seed)
    p, g, d = s["p"].double(), s["g"].double(), s["decay"].double()
    t = STEPS + 1
    out = {}
    if case["clip"]:
        norm = torch.linalg.vector_norm(g)
        out["norm"] = norm.view(1)
        if norm > case["clip"]:
            g = g * (case["clip"] / norm)
    if case["bits"] == 8:
        codes = s["m"].double()
        m = (codes.abs() / 127) ** 2 * codes.sign() * s["ms"].double().repeat_interleave(PAD)
        v = (s["v"].double() / 255) ** 4 * s["vs"].double().repeat_interleave(PAD)
    else:
        m, v = s["m"].double(), s["v"].double()
    m = torch.lerp(m, g, 1 - B1)
    v = torch.lerp(v, g ** 2, 1 - B2)
    # sqrt(v / (1 - b2^t)) + eps, with both corrections taken out of the quotient
    size = LR * math.sqrt(1 - B2 ** t) / (1 - B1 ** t)
    out["p"] = p * (1 - LR * d) - size * m / (v.sqrt() + EPS * math.sqrt(1 - B2 ** t))
    if case["bits"] == 8:
        ms, vs = (x.reshape(-1, PAD).abs().max(1).values for x in (m, v))
        wide_m, wide_v = ms.repeat_interleave(PAD), vs.repeat_interleave(PAD)
        code = torch.where(wide_m > 0, 127 * (m.abs() / wide_m) ** 0.5, 0.0).round() * m.sign()
        part = torch.where(wide_v > 0, v / wide_v, 0.0)
        floor = torch.minimum(torch.floor(255 * part ** 0.25), torch.full_like(part, 254.0))
        chance = (part - (floor / 255) ** 4) / (((floor + 1) / 255) ** 4 - (floor / 255) ** 4)
        grain = _bits16(s["seed"], t, m.numel()).double() / 65536
        b = torch.where(grain < chance, floor + 1, floor)
        b = torch.where((b == 0) & (v > 0), 1.0, b)
        out |= dict(m=(code / 127) ** 2 * code.sign() * wide_m, v=(b / 255) ** 4 * wide_v, m_scale=ms, v_scale=vs)
    else:
        out |= dict(m=m, v=v)
    return out


def _exact_few(x, s):
    """Rows of few logits: every pair compared."""
    n = x.shape[1]
    at = torch.arange(n, device="cuda")
    first = (x[:, None, :] > x[:, :, None]) | ((x[:, None, :] == x[:, :, None]) & (at < at[:, None]))  # j before i
    top = x.max(1, keepdim=True).values
    live = x > -math.inf
    w = torch.where(live, torch.exp((x - top) / s["temperature"].double()[:, None]), 0.0)
    k = s["top_k"][:, None]
    w = torch.where((first.sum(2) < k) | (k == 0), w, 0.0)
    p = s["top_p"].double()[:, None]
    ahead = torch.where(first, w[:, None, :], 0.0).sum(2)
    keep = live & (w >= s["min_p"].double()[:, None]) & ((ahead < p * w.sum(1, keepdim=True)) | (p >= 1))
    w = torch.where(keep, w, 0.0) / torch.where(keep, w, 0.0).sum(1, keepdim=True)
    below = torch.where(at <= at[:, None], w[:, None, :], 0.0).sum(2)
    hit = ((below > s["u"].double()[:, None]) & (w > 0)).int()
    index, any_ = hit.argmax(1), hit.any(1)
    return dict(index=torch.where(any_, index, -1).int(), prob=torch.where(any_, w.gather(1, index[:, None])[:, 0], 0.0))


def _exact_sample(case, seed):
    s = _prepare_sample(case, seed)
    x = s["x"].double()
    if s["mask"] is not None:
        x[s["mask"] != 0] = -math.inf
    rows, n = x.shape
    if rows * n * n <= 200_000_000:
        return _exact_few(x, s)
    if rows > 1024:
        return None
    index, prob = torch.full((rows,), -1, dtype=torch.int32), torch.zeros(rows, dtype=torch.float64)
    for r in range(rows):
        live = torch.nonzero(x[r] > -math.inf).view(-1)
        if not live.numel():
            continue
        t = float(s["temperature"][r])
        w = torch.exp((x[r, live] - x[r, live].max()) / t)
        order = torch.argsort(-x[r, live], stable=True)
        if 0 < int(s["top_k"][r]) < order.numel():
            order = order[:int(s["top_k"][r])]
        if float(s["top_p"][r]) < 1:
            mass = torch.cumsum(w[order], 0)
            order = order[:int((mass < float(s["top_p"][r]) * mass[-1]).sum()) + 1]
        order = order[w[order] >= float(s["min_p"][r])].sort().values
        mass = torch.cumsum(w[order], 0)
        at = min(int(torch.searchsorted(mass, float(s["u"][r]) * mass[-1], right=True)), order.numel() - 1)
        index[r] = int(live[order[at]])
        prob[r] = float(w[order[at]] / mass[-1])
    return dict(index=index, prob=prob)


def exact(case, seed):
    return _exact_adamw(case, seed) if case["op"] == "adamw" else _exact_sample(case, seed)
