"""The mixture-of-experts layer on the GPU against the plain 64-bit form.

Bound on y (mx4_reference.moe): fp32 sums of K products lose at most gamma(K) = 2 K 2^-24 relative
to the sum of magnitudes for 16-bit weights (each mma step of 16 may truncate 17 2^-24 of what it
adds: 1.07 K 2^-24 in all, and the parts of up to eight warps are added once more), less for
four-bit ones; h is rounded once to the layer's type (eps/2 relative) and y once more.
For more than eight tokens h goes on as three e4m3 pieces (four-bit weights) or two values of the
type, and tokens as pieces too: within 2^-13, far below the type's rounding that the bound has for h.
Inputs have few bits, so that the 64-bit logits of kernel and plain form are the same number
and ties are real ties.
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


def gamma(k):
    return (2 * k + 32) * 2.0 ** -24


def layer(seed, tokens, experts, hidden, inter, dtype, four_bit):
    r = np.random.RandomState(seed)

    def few_bits(shape, scale):
        return np.round(r.randn(*shape) * 16) / 16 * scale
    d = {"x": torch.from_numpy(few_bits((tokens, hidden), 1.0)).to(dtype).cuda(),
         "router": torch.from_numpy(few_bits((experts, hidden), 2.0 ** -round(np.log2(hidden) / 2))).to(dtype).cuda()}
    v = {}
    for name, rows, cols in (("gate", inter, hidden), ("up", inter, hidden), ("down", hidden, inter)):
        m = r.randn(experts, rows, cols) * cols ** -0.5
        if four_bit:
            c, s = R.quantize(m.reshape(-1, cols))
            c, s = c.reshape(experts, rows, -1), s.reshape(experts, rows, -1)
            d[name], d[name + "_scales"] = torch.from_numpy(c).cuda(), torch.from_numpy(s).cuda()
            v[name] = R.values(c, s, cols)
        else:
            d[name] = torch.from_numpy(m).to(dtype).cuda()
            v[name] = np64(d[name])
    return d, v


def call(d, topk, renormalize=True, workspace=None, **out):
    tokens, inter = d["x"].shape[0], d["gate"].shape[1]
    y = torch.full(d["x"].shape, float("nan"), dtype=d["x"].dtype, device="cuda")
    ids = torch.full((tokens, topk), -1, dtype=torch.int32, device="cuda")
    w = torch.full((tokens, topk), float("nan"), device="cuda")
    ws = S.moe_workspace(tokens, d["router"].shape[0], topk, inter) if workspace is None else workspace
    S.moe_out(d["x"], d["router"], d["gate"], d["up"], d["down"], y, ws, topk, renormalize=renormalize,
              gate_scales=d.get("gate_scales"), up_scales=d.get("up_scales"), down_scales=d.get("down_scales"),
              ids=ids, weights=w)
    assert binding.device_error() == 0
    return y, ids, w


def check(d, v, topk, renormalize, got):
    y, ids, w = got
    dtype = d["x"].dtype
    f = torch.finfo(dtype)
    want, bound, wids, ww = R.moe(np64(d["x"]), np64(d["router"]), v["gate"], v["up"], v["down"], topk, renormalize,
                                  f.eps / 2, gamma)
    assert np.array_equal(ids.cpu().numpy(), wids)
    # softmax in fp32: expf (2 ulp), a sum of at most 256 terms in a tree of 14 adds, one division, and the
    # rounding of the logits' difference to fp32 (2^-24 of at most 32 here)
    assert (np.abs(np64(w) - ww) <= 2.0 ** -18 * ww + 1e-30).all()
    bound = bound + 2.0 ** -18 * np.abs(want)
    limit = bound + np.maximum((np.abs(want) + bound) * f.eps / 2, f.tiny * f.eps / 2)
    err = np.abs(np64(y) - want)
    assert (err <= limit).all(), float(np.nanmax(err / limit))


@pytest.mark.parametrize("kind", ["fp16", "bf16"])
@pytest.mark.parametrize("four_bit", [False, True])
@pytest.mark.parametrize("tokens,experts,topk,hidden,inter", [
    (1, 1, 1, 1, 1), (1, 2, 1, 32, 16), (1, 8, 2, 64, 96), (2, 4, 4, 33, 31), (3, 5, 2, 130, 70), (8, 8, 2, 128, 160),
    (9, 16, 3, 64, 40), (16, 12, 4, 72, 100), (17, 3, 2, 96, 48), (33, 40, 8, 64, 24), (64, 8, 2, 96, 129),
    (64, 256, 16, 32, 16), (1, 8, 2, 512, 1376), (9, 4, 2, 128, 128), (12, 8, 3, 256, 384), (33, 4, 2, 384, 256),
    (64, 2, 2, 256, 640), (20, 16, 4, 640, 128), (64, 32, 8, 128, 200), (40, 3, 1, 136, 1032)])
def test_layer(kind, four_bit, tokens, experts, topk, hidden, inter):
    d, v = layer(tokens + experts, tokens, experts, hidden, inter, TYPES[kind], four_bit)
    for renormalize in (True, False):
        check(d, v, topk, renormalize, call(d, topk, renormalize))


def test_all_tokens_to_one_expert_and_ties():
    d, v = layer(1, 20, 6, 64, 48, torch.float16, False)
    d["router"].zero_()                       # every logit the same: the lowest indices win
    got = call(d, 3)
    assert got[1].tolist() == [[0, 1, 2]] * 20
    check(d, v, 3, True, got)
    d["router"][4] = 1.0
    d["x"].copy_(d["x"].abs())                # one expert above the rest for every token
    got = call(d, 1)
    assert got[1].tolist() == [[4]] * 20
    check(d, v, 1, True, got)


def test_four_bit_experts_with_more_tokens_than_an_item():
    """Few tokens an expert on average, but every token at the same two experts."""
    d, v = layer(11, 64, 16, 96, 70, torch.bfloat16, True)
    d["router"].zero_()
    check(d, v, 2, True, call(d, 2))
    d, v = layer(12, 19, 12, 160, 33, torch.float16, True)
    d["router"].zero_()
    check(d, v, 1, False, call(d, 1, False))


@pytest.mark.parametrize("four_bit", [False, True])
@pytest.mark.parametrize("tokens,experts,topk,hidden,inter", [
    (64, 64, 8, 64, 2000), (64, 6, 6, 40, 3000), (9, 100, 1, 32, 1500), (50, 30, 5, 2500, 32), (7, 20, 3, 64, 2500),
    (12, 24, 2, 3100, 8)])
def test_many_short_items(four_bit, tokens, experts, topk, hidden, inter):
    """Many items of a stage or two on each SM: every ring goes round item after item."""
    for dtype in (torch.float16, torch.bfloat16):
        d, v = layer(tokens, tokens, experts, hidden, inter, dtype, four_bit)
        first = call(d, topk)
        check(d, v, topk, True, first)
        for _ in range(3):
            assert all(torch.equal(a, b) for a, b in zip(call(d, topk), first))


@pytest.mark.parametrize("hidden", [8192, 8200])
@pytest.mark.parametrize("tokens,experts", [(12, 3), (10, 12)])
def test_long_four_bit_tokens(hidden, tokens, experts):
    """Up to the length whose pieces the workspace holds, and beyond it."""
    for dtype in (torch.float16, torch.bfloat16):
        d, v = layer(hidden, tokens, experts, hidden, 40, dtype, True)
        check(d, v, 2, True, call(d, 2))


def test_misaligned_four_bit_layer():
    """Scales and tokens off a word, a short last block, for few and for more tokens."""
    for tokens in (3, 13):
        d, v = layer(13, tokens, 4, 104, 72, torch.float16, True)
        for name in ("gate_scales", "up_scales", "down_scales", "router", "x"):
            room = torch.zeros(d[name].numel() + 1, dtype=d[name].dtype, device="cuda")
            room[1:] = d[name].flatten()
            d[name] = room[1:].view_as(d[name])
        check(d, v, 2, True, call(d, 2))


def test_few_and_more_tokens_share_a_workspace_and_graphs():
    """One workspace for both sizes of batch in turn; two captured graphs with a workspace each,
    replayed on two streams at once."""
    sets = [layer(30 + t, t, 8, 128, 96, torch.float16, q)[0] for t, q in ((4, True), (24, True), (24, False))]
    ws = S.moe_workspace(24, 8, 2, 96)
    first = [call(d, 2, workspace=ws) for d in sets]
    for _ in range(2):
        for d, want in zip(sets, first):
            assert all(torch.equal(a, b) for a, b in zip(call(d, 2, workspace=ws), want))
    graphs, outs = [], []
    for _ in range(2):
        own = S.moe_workspace(24, 8, 2, 96)
        y = [torch.zeros_like(d["x"]) for d in sets]
        g = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(g):
            for d, t in zip(sets, y):
                S.moe_out(d["x"], d["router"], d["gate"], d["up"], d["down"], t, own, 2,
                          **{k: d[k] for k in d if k.endswith("_scales")})
        graphs.append((g, own))
        outs.append(y)
    streams = [torch.cuda.Stream() for _ in graphs]
    for _ in range(5):
        for stream, (g, _) in zip(streams, graphs):
            with torch.cuda.stream(stream):
                g.replay()
    torch.cuda.synchronize()
    for y in outs:
        assert all(torch.equal(t, want[0]) for t, want in zip(y, first))
    assert binding.device_error() == 0


@pytest.mark.parametrize("tokens,hidden,four_bit", [(4, 64, False), (4, 64, True), (12, 128, False), (12, 128, True)])
def test_non_finite_tokens(tokens, hidden, four_bit):
    """A NaN or infinite value makes its token NaN or infinite and leaves the others as they are."""
    d, v = layer(12, tokens, 5, hidden, 128, torch.float16, four_bit)
    clean = call(d, 2)
    d["x"][1, 3], d["x"][3, 40] = float("nan"), float("inf")
    y, ids, w = call(d, 2)
    assert not torch.isfinite(y[1]).any() and not torch.isfinite(y[3]).any()
    for t in [i for i in range(tokens) if i not in (1, 3)]:
        # rows of h move with the others' selections, sums do not
        assert torch.equal(y[t], clean[0][t]) and torch.equal(ids[t], clean[1][t]) and torch.equal(w[t], clean[2][t])


def test_non_finite_logits():
    """A NaN logit is selected first and makes its token NaN; other tokens stay as they are."""
    d, v = layer(2, 4, 5, 64, 32, torch.bfloat16, False)
    clean = call(d, 2)
    d["x"][1, 3] = float("nan")
    y, ids, w = call(d, 2)
    assert ids[1].tolist() == [0, 1] and torch.isnan(w[1]).all() and torch.isnan(y[1]).all()
    for t in (0, 2, 3):
        assert torch.equal(y[t], clean[0][t]) and torch.equal(ids[t], clean[1][t]) and torch.equal(w[t], clean[2][t])
    # an expert masked by the type's lowest value, and one by -inf, are never taken while others remain
    d, v = layer(3, 4, 4, 64, 32, torch.float16, False)
    d["x"][:, 0] = 1.0
    d["router"][:, 0] = 0.0
    d["router"][0, 0] = torch.finfo(torch.float16).min
    d["router"][2, 0] = float("-inf")
    y, ids, w = call(d, 2)
    assert set(ids.flatten().tolist()) == {1, 3} and torch.isfinite(y).all()
    check(d, v, 2, True, (y, ids, w))


def test_workspace_reuse_spaced_rows_and_repeats():
    """One workspace for calls of different sizes; the same bits each time; nothing written beyond y."""
    ws = S.moe_workspace(64, 64, 8, 256)
    a = layer(4, 5, 8, 128, 96, torch.float16, False)
    b = layer(5, 33, 40, 64, 129, torch.float16, True)
    first = call(a[0], 2, workspace=ws)
    check(*b, 8, False, call(b[0], 8, False, workspace=ws))
    for _ in range(3):
        again = call(a[0], 2, workspace=ws)
        assert all(torch.equal(p, q) for p, q in zip(first, again))
    wide = torch.full((5, 300), float("nan"), dtype=torch.float16, device="cuda")
    for off in (8, 3):  # rows on 16 bytes, and not
        wide[:, off:off + 128] = a[0]["x"]
        d = dict(a[0], x=wide[:, off:off + 128])
        room = torch.full((7, 128), 5.0, dtype=torch.float16, device="cuda")
        S.moe_out(d["x"], d["router"], d["gate"], d["up"], d["down"], room[1:6], ws, 2)
        assert torch.equal(room[1:6], first[0]) and (room[0] == 5).all() and (room[6] == 5).all()
        wide.fill_(float("nan"))


def test_misaligned_weights():
    d, v = layer(6, 3, 4, 64, 40, torch.float16, False)
    for name in ("router", "gate", "up", "down"):
        room = torch.zeros(d[name].numel() + 1, dtype=torch.float16, device="cuda")
        room[1:] = d[name].flatten()
        d[name] = room[1:].view_as(d[name])
    check(d, v, 2, True, call(d, 2))


def test_graph_replays_and_streams():
    d, v = layer(7, 6, 8, 128, 96, torch.bfloat16, True)
    ws, ws2 = (S.moe_workspace(6, 8, 2, 96) for _ in range(2))
    y = torch.empty_like(d["x"])
    args = (d["x"], d["router"], d["gate"], d["up"], d["down"])
    scales = {k: d[k] for k in ("gate_scales", "up_scales", "down_scales")}
    S.moe_out(*args, y, ws, 2, **scales)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        for _ in range(3):
            S.moe_out(*args, y, ws, 2, **scales)
    for seed in range(3):
        d["x"].copy_(layer(20 + seed, 6, 8, 128, 96, torch.bfloat16, True)[0]["x"])
        y.zero_()
        g.replay()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        z = torch.empty_like(y)
        with torch.cuda.stream(side):
            S.moe_out(*args, z, ws2, 2, **scales)
        torch.cuda.synchronize()
        assert torch.equal(y, z) and torch.equal(y, S.moe(*args, 2, **scales))
    assert binding.device_error() == 0


def test_quantised_experts_together():
    """A 16-bit layer, its experts rounded to four bits by mx4_quantize: the layer on the codes equals
    the layer on the values read back, within the bound, and one expert's product equals mx4_project's."""
    d, _ = layer(8, 4, 4, 160, 96, torch.float16, False)
    q = dict(d)
    v = {}
    for name in ("gate", "up", "down"):
        q[name], q[name + "_scales"] = S.mx4_quantize(d[name])
        v[name] = np64(S.mx4_dequantize(q[name], q[name + "_scales"], d[name].shape[-1], torch.float32))
    check(q, v, 2, True, call(q, 2))
    one = {k: (t[:1].contiguous() if k != "x" else t) for k, t in q.items()}
    y, ids, w = call(one, 1)
    assert (w == 1).all() and (ids == 0).all()
    g = S.mx4_project(q["x"], q["gate"][0], q["gate_scales"][0], dtype=torch.float32)
    u = S.mx4_project(q["x"], q["up"][0], q["up_scales"][0], dtype=torch.float32)
    h = (g / (1 + torch.exp(-g)) * u).half()
    z = S.mx4_project(h, q["down"][0], q["down_scales"][0])
    # the same sums in another split: h may differ by one rounding, y by its effect
    scale = np.abs(v["down"][0]) @ np.abs(np64(h)).T
    limit = scale.T * 2.0 ** -10 + np.abs(np64(z)) * 2.0 ** -10
    assert (np.abs(np64(y) - np64(z)) <= limit).all()


def test_refusals():
    d, _ = layer(9, 2, 4, 64, 32, torch.float16, False)
    y, ws = torch.empty_like(d["x"]), S.moe_workspace(2, 4, 2, 32)
    good = [d["x"], d["router"], d["gate"], d["up"], d["down"], y, ws, 2]

    def bad(i, value, **kw):
        a = list(good)
        a[i] = value
        with pytest.raises(RuntimeError):
            S.moe_out(*a, **kw)
    bad(0, d["x"].float()), bad(0, d["x"][0]), bad(1, d["router"][:, :32]), bad(1, d["router"].bfloat16())
    bad(2, d["gate"][:3]), bad(3, d["up"].transpose(1, 2)), bad(4, d["down"][:, :, :16]), bad(5, y[:1])
    bad(6, ws[:256]), bad(7, 0), bad(7, 5), bad(6, ws.cpu())
    bad(5, d["x"])                                         # y over x
    q, s = S.mx4_quantize(d["gate"])
    bad(2, q, gate_scales=s)
    bad(0, d["x"], ids=torch.empty((2, 2), dtype=torch.int64, device="cuda"))
    bad(0, d["x"], weights=torch.empty((2, 3), device="cuda"))
    S.moe_out(*good)
    S.moe_out(d["x"][:0], d["router"], d["gate"], d["up"], d["down"], y[:0], ws, 2)
