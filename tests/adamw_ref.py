"""AdamW in 64 bits with the error bounds of an fp32 evaluation (test infrastructure).

All bounds count roundings: U = 2^-24 is half a step of fp32, relative to the value.
"""
import numpy as np

import devrng

U = 2.0 ** -24
HALF = {"f32": U, "bf16": 2.0 ** -8, "f16": 2.0 ** -11}
BLK = 256


def places(sizes):
    """(starts, total) of the state layout."""
    starts, at = [], 0
    for s in sizes:
        starts.append(at)
        at += -(-s // BLK) * BLK
    return starts, at


def bits16(seed, t, total):
    key = devrng.splitmix64(seed ^ ((t * 0xD1B54A32D192ED03) & devrng.M64))
    z = (np.arange(-(-total // 4), dtype=np.uint64) ^ np.uint64(key)) + np.uint64(0x9E3779B97F4A7C15)
    z = (z ^ (z >> np.uint64(30))) * np.uint64(0xBF58476D1CE4E5B9)
    z = (z ^ (z >> np.uint64(27))) * np.uint64(0x94D049BB133111EB)
    z = z ^ (z >> np.uint64(31))
    return np.stack([(z >> np.uint64(16 * j)) & np.uint64(0xFFFF) for j in range(4)], 1).reshape(-1)[:total].astype(np.float64)


def m_values(codes, scale):
    a = codes.astype(np.float64)
    return a * np.abs(a) / 127.0 ** 2 * np.repeat(scale.astype(np.float64), BLK)


def v_values(codes, scale):
    return (codes.astype(np.float64) / 255.0) ** 4 * np.repeat(scale.astype(np.float64), BLK)


def norm(g, scale):
    return float(np.sqrt(np.sum((g.astype(np.float64) * scale) ** 2)))


class Step:
    """One step on flat arrays in the state layout (zeros between tensors). p, g: the stored values;
    m, v: the old moments' values. Gives the new m, v, p in 64 bits and how far an fp32 evaluation
    may be off: em, ev, ep (before p's own rounding)."""

    def __init__(self, p, g, m, v, t, *, lr, b1, b2, eps, wd, scale=1.0, max_norm=0.0, state_bits=32):
        p, g, m, v = (np.asarray(x, np.float64) for x in (p, g, m, v))
        lr, eps, wd = float(np.float32(lr)), float(np.float32(eps)), np.float32(wd).astype(np.float64)
        self.norm = norm(g, scale)
        c = max_norm / self.norm if max_norm and self.norm > max_norm else 1.0
        gp = g * (float(np.float32(scale)) * c)
        # g': the product's and the factor's rounding (2 U). Old values of 8-bit states: m 4 U (constant,
        # two products), v 12 U ((b / 255): 2 U,
        # squared 5 U, squared again 11 U, times the scale)
        old_m, old_v = (0, 0) if state_bits == 32 else (4, 12)
        self.m = b1 * m + (1 - b1) * gp
        self.em = U * ((3 + old_m) * np.abs(b1 * m) + 5 * np.abs((1 - b1) * gp)) + 1e-44
        self.v = b2 * v + (1 - b2) * gp * gp
        self.ev = U * ((3 + old_v) * b2 * v + 8 * (1 - b2) * gp * gp) + 1e-44
        c1, c2 = 1 / (1 - b1 ** t), 1 / (1 - b2 ** t)
        root = np.sqrt(self.v * c2)
        # the root's error: ev through its slope, 3 U of its own; at v = 0 the whole of sqrt(ev)
        eroot = np.sqrt((self.v + self.ev) * c2) - np.sqrt(np.maximum(self.v - self.ev, 0) * c2) + 3 * U * root
        den = root + eps
        step = self.m * c1 / den
        self.estep = (self.em * c1 + np.abs(self.m) * c1 * (eroot + U * den) / den) / np.maximum(den - eroot - U * den, eps * 0.5) \
            + 4 * U * np.abs(step)
        self.p = p - lr * (step + wd * p)
        self.ep = lr * (self.estep + 3 * U * np.abs(wd * p) + 3 * U * np.abs(step + wd * p)) + U * np.abs(self.p) + U * np.abs(p)

    def codes_ok(self, a, ms, b, vs, rand):
        """Whether codes a (int8), b (uint8) and scales are those of the new moments: every code must
        be one that some m, v within the error bounds rounds to."""
        m, v = self.m.reshape(-1, BLK), self.v.reshape(-1, BLK)
        em, ev = self.em.reshape(-1, BLK), self.ev.reshape(-1, BLK)
        ms, vs = ms.astype(np.float64)[:, None], vs.astype(np.float64)[:, None]
        top_m, top_v = np.abs(m).max(1, keepdims=True), v.max(1, keepdims=True)
        assert np.all(np.abs(ms - top_m) <= em.max(1, keepdims=True) + U * top_m), "m scales"
        assert np.all(np.abs(vs - top_v) <= ev.max(1, keepdims=True) + U * top_v), "v scales"
        a, b, rand = (x.reshape(-1, BLK).astype(np.float64) for x in (a, b, rand))

        def m_code(x):   # monotone in x
            r = np.where(ms > 0, np.abs(x) / np.where(ms > 0, ms, 1), 0)
            return np.sign(x) * 127 * np.sqrt(r)
        # three roundings of the quotient, root and product (the quotient's halves in the root): 3 U of 127
        slack = 3 * U * 127
        assert np.all((a >= np.rint(m_code(m - em) - slack)) & (a <= np.rint(m_code(m + em) + slack))), "m codes"

        def v_code(part, r):   # monotone: up in part, down in r
            low = np.minimum(np.floor(255 * np.maximum(part, 0) ** 0.25), 254)
            lo, hi = (low / 255) ** 4, ((low + 1) / 255) ** 4
            return low + (r < (part - lo) / (hi - lo) * 65536)
        base = np.where(vs > 0, vs, 1)
        # the chance's own error: levels 11 U each, times level / (hi - lo) <= b / 4: 22 U * 64, in 65536ths: 5.5
        lowest = v_code((v - ev) / base * (1 - 4 * U), rand + 8)
        highest = v_code((v + ev) / base * (1 + 4 * U), rand - 8)
        # a quotient next to a level's edge may be floored to either side
        lowest = np.minimum(lowest, v_code((v - ev) / base * (1 - 64 * U), rand + 8))
        highest = np.maximum(highest, v_code((v + ev) / base * (1 + 64 * U), rand - 8))
        live = v > 0
        lowest, highest = np.where(live, np.maximum(lowest, 1), lowest), np.where(live, np.maximum(highest, 1), highest)
        assert np.all((b >= lowest) & (b <= highest)), "v codes"
        assert np.all(b[~live & (ev <= 1e-44)] == 0), "v codes of nothing"
