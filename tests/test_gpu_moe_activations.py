"""What the expert layer keeps of h = SiLU(gate x) * (up x) between its two products.

h leaves the gate phase in fp32's range and is held as
  fp16         two values of the type after a power of two of its row: within 2^-22 of itself and
               2^-38 of its row's largest (the remainder's half step, 2^-25, beside [2^14, 2^15))
  bf16         two values: within 2^-16 (2^-8 of what a rounding to 2^-8 left)
  four bits, more than eight tokens: three e4m3 pieces, within 2^-14 of the largest of its block of
               32 (largest in [128, 256): a step of 16 there, so a piece leaves 8, twice times 32)
"""
import numpy as np
import pytest
import torch

import mx4_reference as R
import swiglu_b200 as S
from swiglu_b200 import binding

pytestmark = pytest.mark.gpu
TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}


def np64(t):
    return t.double().cpu().numpy()


def put(dtype, four_bit, x, router, **matrices):
    """A layer's tensors, and the values that they hold."""
    d = {"x": torch.from_numpy(x).to(dtype).cuda(), "router": torch.from_numpy(router).to(dtype).cuda()}
    v = {"x": np64(d["x"]), "router": np64(d["router"])}
    for name, m in matrices.items():
        if four_bit:
            c, s = R.quantize(m.reshape(-1, m.shape[-1]))
            c, s = c.reshape(*m.shape[:2], -1), s.reshape(*m.shape[:2], -1)
            d[name], d[name + "_scales"] = torch.from_numpy(c).cuda(), torch.from_numpy(s).cuda()
            v[name] = R.values(c, s, m.shape[-1])
        else:
            d[name] = torch.from_numpy(m).to(dtype).cuda()
            v[name] = np64(d[name])
    return d, v


def call(d, topk, workspace=None):
    tokens, inter = d["x"].shape[0], d["gate"].shape[1]
    y = torch.full_like(d["x"], float("nan"))
    ids = torch.full((tokens, topk), -1, dtype=torch.int32, device="cuda")
    ws = S.moe_workspace(tokens, d["router"].shape[0], topk, inter) if workspace is None else workspace
    S.moe_out(d["x"], d["router"], d["gate"], d["up"], d["down"], y, ws, topk, ids=ids,
              **{k: d[k] for k in d if k.endswith("_scales")})
    assert binding.device_error() == 0
    return y, ids


def kept(h, dtype, four_bit):
    """How far the held h may be from the fp32 one (rows of h)."""
    if four_bit and h.shape[0] > 8:
        pad = np.zeros((h.shape[0], -(-h.shape[1] // 32) * 32))
        pad[:, :h.shape[1]] = np.abs(h)
        top = pad.reshape(h.shape[0], -1, 32).max(2).repeat(32, 1)[:, :h.shape[1]]
        return 2.0 ** -14 * top
    if dtype == torch.bfloat16:
        return 2.0 ** -16 * np.abs(h) + 2.0 ** -133
    return 2.0 ** -22 * np.abs(h) + 2.0 ** -38 * np.abs(h).max(1, keepdims=True)


def gamma(k):
    """Sums of K products relative to their magnitudes: each step of 16 may truncate 17 2^-24, the parts
    of up to 16 warps and a cluster's are added once more."""
    return (2 * k + 40) * 2.0 ** -24


def one_expert_each(v, dtype, four_bit, ids):
    """(y, bound) for topk 1, whose weight is exactly 1."""
    ids = ids.cpu().numpy()[:, 0]
    x = v["x"]
    gk, gi = gamma(x.shape[1]), gamma(v["down"].shape[2])
    g = np.stack([v["gate"][e] @ t for e, t in zip(ids, x)])
    u = np.stack([v["up"][e] @ t for e, t in zip(ids, x)])
    dg = gk * np.stack([np.abs(v["gate"][e]) @ np.abs(t) for e, t in zip(ids, x)])
    du = gk * np.stack([np.abs(v["up"][e]) @ np.abs(t) for e, t in zip(ids, x)])
    with np.errstate(over="ignore"):
        silu = g / (1 + np.exp(-g))
    h = silu * u
    # |silu'| <= 1.1; silu to 2^-21 relative in fp32, the product rounded once
    dh = 1.1 * dg * np.abs(u) + np.abs(silu) * du + 1.1 * dg * du + 2.0 ** -20 * np.abs(h)
    dh = dh + kept(np.abs(h) + dh, dtype, four_bit)
    y = np.stack([v["down"][e] @ t for e, t in zip(ids, h)])
    bound = np.stack([np.abs(v["down"][e]) @ t for e, t in zip(ids, dh)])
    return y, bound + gi * np.stack([np.abs(v["down"][e]) @ t for e, t in zip(ids, np.abs(h) + dh)]), h


def within(y, want, bound):
    f = torch.finfo(y.dtype)
    limit = bound + np.maximum((np.abs(want) + bound) * f.eps / 2, f.tiny * f.eps / 2)
    err = np.abs(np64(y) - want)
    assert np.isfinite(err).all(), "not finite"
    assert (err <= limit).all(), float((err / limit).max())


def spread(seed, tokens, dtype, four_bit, regime, hidden=64, inter=96):
    """h of the asked magnitude and y within fp16's range."""
    r = np.random.RandomState(seed)
    gate, up, down = {"large": (2.0 ** 6, 2.0 ** 6, 2.0 ** -12), "small": (2.0 ** -11, 2.0 ** -14, 2.0 ** 9),
                      "mixed": (1.0, 1.0, 2.0 ** -6)}[regime]
    x = r.randn(tokens, hidden)
    if regime == "mixed":  # neighbouring tokens' h a factor of up to 2^26 apart
        x = x * 2.0 ** (r.randint(-8, 6, (tokens, 1)))
    return put(dtype, four_bit, x, r.randn(3, hidden), gate=r.randn(3, inter, hidden) * gate,
               up=r.randn(3, inter, hidden) * up, down=r.randn(3, hidden, inter) * down)


@pytest.mark.parametrize("kind", ["fp16", "bf16"])
@pytest.mark.parametrize("four_bit", [False, True])
@pytest.mark.parametrize("tokens", [1, 8, 9, 40])
@pytest.mark.parametrize("regime", ["large", "small", "mixed"])
def test_range_of_activations(kind, four_bit, tokens, regime):
    """Beyond 65504, near fp16's least values, and both in one batch: y is as close as h's bits allow, in
    a batch of eight as in one of nine."""
    d, v = spread(3, tokens, TYPES[kind], four_bit, regime)
    y, ids = call(d, 1)
    want, bound, h = one_expert_each(v, TYPES[kind], four_bit, ids)
    if regime == "large":
        assert np.abs(h).max(1).min() > 65504 and np.abs(want).max() < 65504
    if regime == "small":
        assert np.abs(h).max() < 2.0 ** -14 and np.abs(want).max() > 2.0 ** -12
    within(y, want, bound)


@pytest.mark.parametrize("kind", ["fp16", "bf16"])
@pytest.mark.parametrize("four_bit", [False, True])
@pytest.mark.parametrize("tokens", [1, 8, 9, 33])
def test_remainder_of_activations(kind, four_bit, tokens):
    """Rows of down that cancel the rounded h, so that y consists of what the rounding left.

    h of places i and i + 32 have one gate row and up rows 2^-6 apart; a row of down takes their
    difference. x is -1, 0 or 1 and the matrices hold codes of two blocks, so that every partial sum
    of gate and up is a multiple of 2^-7 below 2^9 and exact in fp32 in any order. The two places then
    share the computed silu: its error scales y (2^-20), the product of h rounds once (2^-24 |h|)."""
    dtype = TYPES[kind]
    r = np.random.RandomState(5)
    hidden, m = 64, 32
    codes = np.array([.5, 1, 1.5, 2, 3, 4, 6])
    x = r.randint(-1, 2, (tokens, hidden)).astype(np.float64)
    x[:, 0], x[:, 32] = 1, 1
    gate, up, down = (np.zeros((2, 2 * m, hidden)) for _ in range(3))
    down = np.zeros((2, hidden, 2 * m))
    for e in range(2):
        gate[e, :m, :4] = codes[r.randint(0, 7, (m, 4))]
        gate[e, m:] = gate[e, :m]
        up[e, :m, :32] = codes[r.randint(0, 7, (m, 32))] * r.choice([-1, 1], (m, 32))
        up[e, :m, 0] = 6
        up[e, m:] = up[e, :m]
        up[e, m:, 32] = codes[r.randint(0, 7, m)] * 2.0 ** -6
        for row in range(hidden):
            down[e, row, row % m], down[e, row, row % m + m] = 1, -1
    d, v = put(dtype, four_bit, x, r.randn(2, hidden), gate=gate, up=up, down=down)
    assert all(np.array_equal(v[k], w) for k, w in (("gate", gate), ("up", up), ("down", down), ("x", x)))
    y, ids = call(d, 1)
    e = ids.cpu().numpy()[:, 0]
    g, u = np.stack([gate[k] @ t for k, t in zip(e, x)]), np.stack([up[k] @ t for k, t in zip(e, x)])
    h = g / (1 + np.exp(-g)) * u
    want = np.stack([down[k] @ t for k, t in zip(e, h)])
    # of the two places: the product's rounding, what is kept; of their sum in the tensor core: two products
    # of each of up to three parts, a truncation of 17 2^-24 each, and the parts' additions
    dh = 2.0 ** -24 * np.abs(h) + kept(h, dtype, four_bit) + 7 * 17 * 2.0 ** -24 * np.abs(h)
    bound = np.stack([np.abs(down[k]) @ t for k, t in zip(e, dh)]) + 2.0 ** -20 * np.abs(want)
    within(y, want, bound)


def test_calls_of_other_magnitudes_share_a_workspace():
    """Large, small and mixed activations, few and more tokens, routed alone or together, in turn on one
    workspace: the same bits as with a workspace of their own, call after call and in a graph."""
    ws = S.moe_workspace(40, 40, 1, 96)
    sets = []
    for seed, (tokens, regime, four_bit) in enumerate(
            [(1, "large", False), (1, "small", False), (8, "small", True), (8, "large", True), (9, "large", False),
             (9, "small", False), (40, "large", True), (40, "mixed", False), (8, "mixed", False), (1, "small", True)]):
        sets.append(spread(seed, tokens, torch.float16, four_bit, regime)[0])
    # many experts: the router's work is shared, and waits for a barrier of its own
    d = spread(50, 8, torch.float16, False, "small")[0]
    for k in ("router", "gate", "up", "down"):
        d[k] = d[k].repeat(8, *[1] * (d[k].dim() - 1))
    sets.append(d)
    fresh = [call(d, 1) for d in sets]
    r = np.random.RandomState(0)
    for i in list(range(len(sets))) + list(r.randint(0, len(sets), 40)):
        assert all(torch.equal(a, b) for a, b in zip(call(sets[i], 1, ws), fresh[i])), i
    ys = [torch.zeros_like(d["x"]) for d in sets]
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        for d, y in zip(sets, ys):
            S.moe_out(d["x"], d["router"], d["gate"], d["up"], d["down"], y, ws, 1,
                      **{k: d[k] for k in d if k.endswith("_scales")})
    for _ in range(3):
        for y in ys:
            y.zero_()
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(y, f[0]) for y, f in zip(ys, fresh))
    assert binding.device_error() == 0


def test_non_finite_activations_stay_in_their_token():
    """A token whose h is beyond fp32, or NaN, is not finite; its neighbours keep their bits."""
    for tokens in (8, 9):
        for four_bit in (False, True):
            d, _ = spread(9, tokens, torch.float16, four_bit, "mixed")
            clean, ids = call(d, 1)
            d["x"][2, 5] = float("nan")
            d["x"][4, 7] = float("inf")
            y, now = call(d, 1)
            for t in range(tokens):
                if t in (2, 4):
                    assert not torch.isfinite(y[t]).any()
                else:
                    assert torch.equal(y[t], clean[t]) and torch.equal(now[t], ids[t])
