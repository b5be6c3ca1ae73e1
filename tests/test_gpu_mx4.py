"""Four-bit matrices on the GPU against plain 64-bit forms.

Rounding and reading back are exact (whole codes, power-of-two scales), so they are compared
bit for bit; reading back as fp16 rounds what fp16 cannot hold, and is compared with numpy's
rounding of the exact value.

Products with 16-bit tokens sum exact products in fp32. One tensor-core step of k products and the
running sum may lose (k + 2) 2^-24 of the magnitudes it adds (aligned to the largest, truncated);
k is 16 or 32, so K values lose at most 1.125 K 2^-24 of sum|w x|, and the parts of clusters or
warps, bias and residual add at most 76 roundings more. Where a token is split into e4m3 pieces, a
value within 13 binades of its block's largest is exact, and another is off by at most half the
last piece's smallest step: 2^-10 of the piece's unit, which is 2^10 (three pieces, fp16) or
2^5 (two, bf16) below the first's, where the largest is at least 2^7: 2^-27 or 2^-22 of it. Where
fp16 weights are decoded against their row's largest scale, values are exact within 2^36 of it, as
they are for these inputs but where a test says otherwise.
So |out - exact| <= (1.125 K + 76) 2^-24 sum|w x| + d sum over blocks of max|x| sum|w| (+ |bias| +
|residual| in the first sum) + half a step of the output type (eps/2 relative, or half of the
smallest subnormal).

Products of two four-bit matrices: one tensor-core step adds 64 exact products to the running sum
and may lose 66 2^-24 of the magnitudes it adds; the cluster's eight parts, bias and residual
add ten roundings more: |out - exact| <= (1.1 K + 76) 2^-24 sum|w x| + half a step of the output.
"""
import numpy as np
import pytest
import torch

import mx4_reference as R
import swiglu_b200 as S
from swiglu_b200 import binding

pytestmark = pytest.mark.gpu
TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}


def sample(shape, dtype, seed, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * scale).to(dtype).cuda()


def np64(t):
    return t.double().cpu().numpy()


def packed(shape, seed, scale=1.0):
    """A four-bit matrix as the plain form rounds it: (codes, scales) on the GPU, values."""
    x = np.random.RandomState(seed).randn(*shape) * scale
    c, s = R.quantize(x.reshape(-1, shape[-1]))
    c, s = c.reshape(*shape[:-1], -1), s.reshape(*shape[:-1], -1)
    return torch.from_numpy(c).cuda(), torch.from_numpy(s).cuda(), R.values(c, s, shape[-1])


@pytest.mark.parametrize("kind", ["fp16", "bf16", "fp32"])
@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 32), (3, 31), (5, 33), (2, 8), (7, 40), (4, 257), (9, 1030), (65, 96)])
def test_quantize_and_back(kind, rows, cols):
    x = sample((rows, cols), TYPES[kind], rows * 1000 + cols, 3.0)
    codes, scales = S.mx4_quantize(x)
    c, s = R.quantize(np64(x))
    assert np.array_equal(codes.cpu().numpy(), c) and np.array_equal(scales.cpu().numpy(), s)
    back = S.mx4_dequantize(codes, scales, cols, TYPES[kind])
    want = torch.from_numpy(R.values(c, s, cols)).to(TYPES[kind])
    assert torch.equal(back.cpu(), want)
    whole = S.mx4_dequantize(codes, scales, dtype=torch.float32)  # pads read as zeros
    assert whole.shape[1] == -(-cols // 32) * 32 and not whole[:, cols:].any()


def test_quantize_ties_and_extremes():
    e = [0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 7.0, 7.99, 6.01, 4.0, -0.25, -0.24, -5.0, 0.0, -0.0]
    rows = [np.array(e + [0.0] * 16) * 2.0 ** k for k in (-140, -131, -127, -126, -100, 0, 3, 100, 124)]
    rows.append(np.zeros(32))
    rows.append(np.full(32, -0.0))
    rows.append(np.full(32, 2.0 ** -149))
    rows.append(np.full(32, np.finfo(np.float32).max))
    x = torch.from_numpy(np.stack(rows).astype(np.float32))
    bad = x[:1].repeat(3, 1).clone()
    bad[0, 3], bad[1, 31], bad[2, 0] = float("nan"), float("inf"), float("-inf")
    x = torch.cat([x, bad]).cuda()
    for view in (x, torch.nn.functional.pad(x, (1, 0))[:, 1:]):  # aligned, and rows off by one value
        codes, scales = S.mx4_quantize(view)
        c, s = R.quantize(np64(x))
        assert np.array_equal(scales.cpu().numpy(), s) and np.array_equal(codes.cpu().numpy(), c)
        back = S.mx4_dequantize(codes, scales, 32, torch.float32).cpu()
        want = torch.from_numpy(R.values(c, s, 32)).float()
        assert torch.equal(torch.isnan(back), torch.isnan(want))
        assert torch.equal(back[:-3], want[:-3]) and torch.isnan(back[-3:]).all()


def test_every_code_and_scale_reads_back():
    codes = torch.arange(256, dtype=torch.uint8).repeat(256, 1).view(256, 16, 16).reshape(256, 256)
    scales = torch.arange(256, dtype=torch.uint8).view(256, 1).repeat(1, 16)
    exact = R.values(codes.numpy(), scales.numpy(), 512)
    for kind in TYPES.values():
        with np.errstate(over="ignore"):
            want = torch.from_numpy(exact.astype(np.float32)).to(kind)  # one rounding: fp32 holds all but the largest
        for cols in (512, 511):
            got = S.mx4_dequantize(codes.cuda(), scales.cuda(), cols, kind).cpu()
            w = want[:, :cols]
            assert torch.equal(torch.isnan(got), torch.isnan(w))
            assert torch.equal(got[~torch.isnan(w)], w[~torch.isnan(w)])


def test_quantize_spaced_rows_three_dims_and_bounds():
    base = sample((6, 200), torch.bfloat16, 1)
    x = base[:, 8:72]
    codes, scales = S.mx4_quantize(x)
    c, s = R.quantize(np64(x))
    assert np.array_equal(codes.cpu().numpy(), c) and np.array_equal(scales.cpu().numpy(), s)
    out = torch.full((6, 200), 7.0, dtype=torch.bfloat16, device="cuda")
    S.mx4_dequantize_out(codes, scales, out[:, 8:72])
    assert torch.equal(out[:, 8:72].cpu().double(), torch.from_numpy(R.values(c, s, 64)))
    assert (out[:, :8] == 7).all() and (out[:, 72:] == 7).all()
    x3 = sample((2, 3, 45), torch.float16, 2)
    c3, s3 = S.mx4_quantize(x3)
    assert c3.shape == (2, 3, 32) and s3.shape == (2, 3, 2)
    c2, s2 = S.mx4_quantize(x3.view(6, 45))
    assert torch.equal(c3.view(6, -1), c2) and torch.equal(s3.view(6, -1), s2)
    empty = S.mx4_quantize(torch.empty((0, 45), dtype=torch.float16, device="cuda"))
    assert empty[0].shape == (0, 32)


def project_bound(x, w, extra, dtype):
    n = -(-x.shape[1] // 32)
    pad = ((0, 0), (0, n * 32 - x.shape[1]))
    largest = np.abs(np.pad(x, pad)).reshape(x.shape[0], n, 32).max(2)
    weights = np.abs(np.pad(w, pad)).reshape(w.shape[0], n, 32).sum(2)
    pieces = (2.0 ** -27 if dtype == torch.float16 else 2.0 ** -22) * (largest @ weights.T)
    return (1.125 * x.shape[1] + 76) * 2.0 ** -24 * (np.abs(x) @ np.abs(w).T + extra) + pieces


def half_step(v, dtype):
    f = torch.finfo(dtype)
    return np.maximum(np.abs(v) * f.eps / 2, f.tiny * f.eps / 2)


def check_product(got, x, w, bias, residual, dtype):
    kind, x = x.dtype, np64(x)
    want = x @ w.T
    extra = np.zeros_like(want)
    for t in (bias, residual):
        if t is not None:
            want = want + t
            extra = extra + np.abs(t)
    bound = project_bound(x, w, extra, kind)
    err = np.abs(np64(got) - want)
    limit = bound + half_step(np.abs(want) + bound, dtype)
    assert np.isfinite(np64(got)).all() and (err <= limit).all(), float((err / limit).max())


@pytest.mark.parametrize("kind", ["fp16", "bf16"])
@pytest.mark.parametrize("tokens,rows,cols", [
    (1, 1, 1), (1, 32, 128), (1, 33, 31), (2, 16, 32), (3, 65, 130), (8, 48, 1024), (9, 100, 257), (16, 31, 160),
    (17, 512, 96), (33, 40, 72), (64, 64, 544), (65, 17, 33), (130, 96, 1030), (1, 5632, 2048),
    (3, 200, 128), (16, 129, 384), (20, 300, 512), (33, 64, 256), (64, 260, 640), (100, 130, 1024), (513, 65, 128),
    (5, 4100, 2048), (2, 128, 100), (12, 192, 4064), (48, 1000, 512), (200, 5000, 320), (700, 200, 1032)])
def test_project(kind, tokens, rows, cols):
    dtype = TYPES[kind]
    codes, scales, w = packed((rows, cols), rows + cols, cols ** -0.5)
    x = sample((tokens, cols), dtype, tokens)
    bias, residual = sample((rows,), dtype, 3, 0.1), sample((tokens, rows), dtype, 4)
    check_product(S.mx4_project(x, codes, scales), x, w, None, None, dtype)
    check_product(S.mx4_project(x, codes, scales, bias, residual, torch.float32), x, w, np64(bias), np64(residual),
                  torch.float32)
    out = residual.clone()
    S.mx4_project_out(x, codes, scales, out, bias, out)  # in place
    check_product(out, x, w, np64(bias), np64(residual), dtype)


def test_project_views_and_bounds():
    """Tokens in spaced or misaligned rows, scales off a word, outputs between guards."""
    codes, scales, w = packed((40, 160), 5, 0.1)
    wide = sample((5, 400), torch.float16, 6)
    room = torch.zeros(scales.numel() + 1, dtype=torch.uint8, device="cuda")
    room[1:] = scales.flatten()
    odd = room[1:].view_as(scales)
    for x in (wide[:, 8:168], wide[:, 3:163]):
        for s in (scales, odd):
            buf = torch.full((7, 40), 9.0, dtype=torch.float32, device="cuda")
            S.mx4_project_out(x, codes, s, buf[1:6])
            check_product(buf[1:6], x, w, None, None, torch.float32)
            assert (buf[0] == 9).all() and (buf[6] == 9).all()


def test_project_special_values():
    """Scales of 0 and 255, the largest scales, and infinities and NaN among the tokens."""
    cols = 128
    codes = torch.randint(0, 256, (48, cols // 2), dtype=torch.uint8, generator=torch.Generator().manual_seed(1))
    scales = torch.full((48, 4), 127, dtype=torch.uint8)
    scales[0] = 0
    scales[1, 2] = 255
    scales[2] = 200
    scales[3, 1] = 0
    w = R.values(codes.numpy(), scales.numpy(), cols)
    for dtype in (torch.float16, torch.bfloat16):
        x = sample((4, cols), dtype, 2)
        got = np64(S.mx4_project(x, codes.cuda(), scales.cuda(), dtype=torch.float32))
        want = np64(x) @ w.T
        assert np.isnan(got[:, 1]).all()
        keep = [i for i in range(48) if i != 1]
        bound = project_bound(np64(x), w[keep], 0, dtype)
        # the smallest scale's products are subnormal in fp32: half of its smallest step each
        assert (np.abs(got[:, keep] - want[:, keep]) <= bound + half_step(want[:, keep], torch.float32) + cols * 2.0 ** -149).all()
        x[2, 5], x[3, 7] = float("inf"), float("nan")
        got = S.mx4_project(x, codes.cuda(), scales.cuda(), dtype=torch.float32)
        rest = S.mx4_project(x[:2].contiguous(), codes.cuda(), scales.cuda(), dtype=torch.float32)
        assert torch.equal(got[:2].nan_to_num(), rest.nan_to_num()) and torch.isnan(got[3]).all()
        assert not torch.isfinite(got[2]).any()


def test_project_far_binades():
    """Tokens whose values span far more binades than a piece holds, block by block."""
    codes, scales, w = packed((70, 256), 11, 0.1)
    for dtype, low in ((torch.float16, -14), (torch.bfloat16, -100)):
        g = torch.Generator().manual_seed(5)
        e = torch.randint(low, 12, (6, 256), generator=g).double()
        x = (torch.randn((6, 256), generator=g).double() * 2.0 ** e).to(dtype).cuda()
        x[1, 32:64] = 0
        x[2] = torch.finfo(dtype).max / 1e4
        x[3] = torch.finfo(dtype).tiny
        for out in (torch.float32, torch.bfloat16):
            check_product(S.mx4_project(x, codes, scales, dtype=out if out == torch.float32 or dtype == out else None), x, w,
                          None, None, torch.float32 if out == torch.float32 else dtype)


@pytest.mark.parametrize("tokens", [17, 40, 70, 150])
def test_project_misaligned_tokens(tokens):
    """More tokens in rows that do not start on 16 bytes, and rows of ragged length."""
    for dtype in (torch.float16, torch.bfloat16):
        codes, scales, w = packed((140, 256), 5, 0.1)
        wide = sample((tokens, 300), dtype, 6)
        buf = torch.full((tokens + 2, 140), 9.0, dtype=torch.float32, device="cuda")
        S.mx4_project_out(wide[:, 3:259], codes, scales, buf[1:-1])
        check_product(buf[1:-1], wide[:, 3:259], w, None, None, torch.float32)
        assert (buf[0] == 9).all() and (buf[-1] == 9).all()
        codes, scales, w = packed((33, 101), 5, 0.1)
        x = sample((tokens, 101), dtype, 7)
        check_product(S.mx4_project(x, codes, scales), x, w, None, None, dtype)


@pytest.mark.parametrize("rows", [48, 192 * 120])
@pytest.mark.parametrize("tokens", [20, 40])
def test_project_special_values_more_tokens(rows, tokens):
    """Extreme scales and non-finite tokens where W is decoded into 16-bit tiles.

    fp16: a value below 2^-36 of its row's largest scale s is off by at most 6 2^-38 s, so the
    product by at most that times sum|x|. bf16 holds every value of scales up to 252."""
    cols = 128
    codes = torch.randint(0, 256, (rows, cols // 2), dtype=torch.uint8, generator=torch.Generator().manual_seed(1))
    scales = torch.full((rows, 4), 127, dtype=torch.uint8)
    scales[0] = 0
    scales[1, 2] = 255
    scales[2] = 200
    scales[3, 1] = 0
    scales[4] = torch.tensor([127, 91, 90, 85])
    scales[5] = torch.tensor([252, 127, 0, 240])
    scales[6] = 255
    w = R.values(codes.numpy(), scales.numpy(), cols)
    keep = [i for i in range(min(rows, 300)) if i not in (1, 6)]
    largest = np.where(scales.numpy() == 255, 0, scales.numpy()).max(1)[keep].astype(np.int64) - 127
    for dtype in (torch.float16, torch.bfloat16):
        x = sample((tokens, cols), dtype, 2, 2.0 ** -6)
        got = np64(S.mx4_project(x, codes.cuda(), scales.cuda(), dtype=torch.float32))
        assert np.isnan(got[:, [1, 6]]).all()
        want = np64(x) @ w[keep].T
        bound = project_bound(np64(x), w[keep], 0, dtype) + cols * 2.0 ** -149
        if dtype == torch.float16:
            bound = bound + 6 * 2.0 ** -38 * np.exp2(largest)[None] * np.abs(np64(x)).sum(1)[:, None]
        assert (np.abs(got[:, keep] - want) <= bound + half_step(np.abs(want) + bound, torch.float32)).all()
        clean = S.mx4_project(x, codes.cuda(), scales.cuda(), dtype=torch.float32)
        x[2, 5], x[3, 7] = float("inf"), float("nan")
        bad = S.mx4_project(x, codes.cuda(), scales.cuda(), dtype=torch.float32)
        rest = [i for i in range(tokens) if i not in (2, 3)]
        assert torch.equal(bad[rest].nan_to_num(), clean[rest].nan_to_num())
        assert torch.isnan(bad[3]).all() and not torch.isfinite(bad[2]).any()


@pytest.mark.parametrize("cols", [32, 64, 100, 128, 192, 200])
def test_project_short_rows_many_tiles(cols):
    """Many tiles of few stages, rows of very different scales: decoding runs far ahead of the epilogue."""
    rows, tokens = 192 * 60, 2000
    rng = np.random.RandomState(cols)
    codes = rng.randint(0, 256, (rows, -(-cols // 32) * 16)).astype(np.uint8)
    if cols % 32:
        codes[:, cols // 2:] = 0
    scales = np.repeat(rng.randint(97, 157, (rows, 1)), -(-cols // 32), axis=1).astype(np.uint8)
    w = R.values(codes, scales, cols)
    for dtype in (torch.float16, torch.bfloat16):
        x = sample((tokens, cols), dtype, 1)
        for _ in range(3):
            got = S.mx4_project(x, torch.from_numpy(codes).cuda(), torch.from_numpy(scales).cuda(), dtype=torch.float32)
            check_product(got, x, w, None, None, torch.float32)


def test_project_refusals():
    codes, scales, _ = packed((8, 64), 1)
    x = sample((2, 64), torch.float16, 1)
    for bad in (lambda: S.mx4_project(x.float(), codes, scales), lambda: S.mx4_project(x[:, :32], codes, scales),
                lambda: S.mx4_project(x, codes[:4], scales), lambda: S.mx4_project(x, codes.cpu(), scales.cpu()),
                lambda: S.mx4_project(x, codes, scales, bias=x[0, :7]),
                lambda: S.mx4_project(x, codes, scales, dtype=torch.bfloat16),
                lambda: S.mx4_project(x.t().contiguous().t(), codes, scales),
                lambda: S.mx4_project(x.requires_grad_(), codes, scales)):
        with pytest.raises(RuntimeError):
            bad()
    assert S.mx4_project(x.detach()[:0], codes, scales).shape == (0, 8)


def test_project_streams_graphs_and_repeats():
    codes, scales, w = packed((96, 512), 8, 0.05)
    x = sample((3, 512), torch.bfloat16, 9)
    want = S.mx4_project(x, codes, scales)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = S.mx4_project(x, codes, scales)
    side.synchronize()
    assert torch.equal(want, again)
    out = torch.empty_like(want)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        S.mx4_project_out(x, codes, scales, out)
    x.copy_(sample((3, 512), torch.bfloat16, 10))
    for _ in range(3):
        out.zero_()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, S.mx4_project(x, codes, scales))


def check_matmul(got, x, w, bias, residual, dtype):
    want, extra = x @ w.T, 0
    for t in (bias, residual):
        if t is not None:
            want, extra = want + t, extra + np.abs(t)
    bound = (1.1 * x.shape[1] + 76) * 2.0 ** -24 * (np.abs(x) @ np.abs(w).T + extra)
    err = np.abs(np64(got) - want)
    limit = bound + half_step(np.abs(want) + bound, dtype)
    assert (err <= limit).all(), float((err / limit).max())


@pytest.mark.parametrize("kind", ["fp16", "bf16"])
@pytest.mark.parametrize("tokens,rows,cols", [
    (1, 1, 1), (1, 128, 256), (2, 33, 31), (7, 129, 130), (16, 256, 512), (17, 100, 1030), (40, 300, 160),
    (64, 128, 2048), (65, 200, 96), (100, 15000, 288), (128, 14300, 70), (128, 130, 640), (129, 192, 256), (200, 385, 1030), (300, 1000, 544),
    (16, 96, 6000), (520, 40, 33)])
def test_matmul(kind, tokens, rows, cols):
    dtype = TYPES[kind]
    xc, xs, x = packed((tokens, cols), tokens, 1.0)
    codes, scales, w = packed((rows, cols), rows + cols, cols ** -0.5)
    bias, residual = sample((rows,), dtype, 3, 0.1), sample((tokens, rows), dtype, 4)
    check_matmul(S.mx4_matmul(xc, xs, codes, scales, dtype=dtype), x, w, None, None, dtype)
    out = residual.clone()
    S.mx4_matmul_out(xc, xs, codes, scales, out, bias, out)  # in place
    check_matmul(out, x, w, np64(bias), np64(residual), dtype)
    buf = torch.full((tokens + 2, rows), 9.0, dtype=dtype, device="cuda")
    S.mx4_matmul_out(xc, xs, codes, scales, buf[1:-1], bias, residual)
    assert torch.equal(buf[1:-1], out) and (buf[0] == 9).all() and (buf[-1] == 9).all()
    assert binding.device_error() == 0


@pytest.mark.parametrize("cols", [32, 256, 300, 600])
def test_matmul_short_rows_many_tiles(cols):
    """Many tiles of one to three stages, rows of very different scales on both sides."""
    rows, tokens = 192 * 60, 2000
    rng = np.random.RandomState(cols)
    n = -(-cols // 32)
    sides = []
    for count in (tokens, rows):
        codes = rng.randint(0, 256, (count, n * 16)).astype(np.uint8)
        codes[:, cols // 2:] = 0
        scales = np.repeat(rng.randint(112, 142, (count, 1)), n, axis=1).astype(np.uint8)
        sides.append((codes, scales, R.values(codes, scales, cols)))
    (xc, xs, x), (wc, ws, w) = sides
    dev = [torch.from_numpy(t).cuda() for t in (xc, xs, wc, ws)]
    for _ in range(2):
        check_matmul(S.mx4_matmul(*dev, dtype=torch.bfloat16), x, w, None, None, torch.bfloat16)


@pytest.mark.parametrize("tokens", [1, 8, 16])
def test_few_tokens_many_short_rows(tokens):
    """Many CTAs of one stage each."""
    codes, scales, w = packed((40000, 72), 3, 0.1)
    for dtype in (torch.float16, torch.bfloat16):
        x = sample((tokens, 72), dtype, 4)
        check_product(S.mx4_project(x, codes, scales), x, w, None, None, dtype)


@pytest.mark.parametrize("tokens", [5, 200])
def test_matmul_special_scales(tokens):
    """NaN scales on either side reach exactly their rows and tokens; extreme scales multiply out;
    misaligned scales take the byte path."""
    rng = np.random.RandomState(1)
    rows, cols = 150, 512
    xc, wc = (rng.randint(0, 256, (n, cols // 2)).astype(np.uint8) for n in (tokens, rows))
    xs, ws = (np.full((n, cols // 32), 127, np.uint8) for n in (tokens, rows))
    ws[3], xs[:, 0] = 10, 130
    ws[7, 5], xs[4, 9] = 255, 255
    x, w = R.values(xc, xs, cols), R.values(wc, ws, cols)
    room = [torch.zeros(t.size + 1, dtype=torch.uint8, device="cuda") for t in (xs, ws)]
    for r, t in zip(room, (xs, ws)):
        r[1:] = torch.from_numpy(t).cuda().flatten()
    dev = [torch.from_numpy(t).cuda() for t in (xc, xs, wc, ws)]
    for sides in (dev, [dev[0], room[0][1:].view(tokens, -1), dev[2], room[1][1:].view(rows, -1)]):
        got = S.mx4_matmul(*sides, dtype=torch.bfloat16)
        assert torch.isnan(got[4]).all() and torch.isnan(got[:, 7]).all()
        t, r = [i for i in range(tokens) if i != 4], [i for i in range(rows) if i != 7]
        check_matmul(got[t][:, r], x[t], w[r], None, None, torch.bfloat16)


def test_matmul_graphs_streams_and_quantised_tokens():
    """Rounding tokens and multiplying, captured together and replayed with new tokens."""
    codes, scales, w = packed((260, 352), 3, 0.06)
    for tokens in (3, 150):
        x = sample((tokens, 352), torch.float16, 4)
        xc, xs = S.mx4_empty(tokens, 352)
        out = torch.empty((tokens, 260), dtype=torch.float16, device="cuda")

        def step():
            S.mx4_quantize_out(x, xc, xs)
            S.mx4_matmul_out(xc, xs, codes, scales, out)
        step()
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            step()
        for seed in range(3):
            x.copy_(sample((tokens, 352), torch.float16, 10 + seed))
            out.zero_()
            g.replay()
            torch.cuda.synchronize()
            c, s = R.quantize(np64(x))
            check_matmul(out, R.values(c, s, 352), w, None, None, torch.float16)
            side = torch.cuda.Stream()
            with torch.cuda.stream(side):
                again = S.mx4_matmul(xc, xs, codes, scales)
            side.synchronize()
            assert torch.equal(again, out)


def test_matmul_refusals():
    xc, xs, _ = packed((4, 64), 1)
    codes, scales, _ = packed((8, 64), 2)
    wide, wide_s, _ = packed((8, 96), 3)
    for bad in (lambda: S.mx4_matmul(xc, xs, wide, wide_s), lambda: S.mx4_matmul(xc, xs, codes, wide_s),
                lambda: S.mx4_matmul(xc, xs, codes, scales, dtype=torch.float32),
                lambda: S.mx4_matmul(xc[:, :16], xs, codes, scales),
                lambda: S.mx4_matmul(xc, xs, codes, scales, bias=torch.zeros(7, device="cuda").half())):
        with pytest.raises(RuntimeError):
            bad()
    assert S.mx4_matmul(xc[:0], xs[:0], codes, scales).shape == (0, 8)


def test_offsets_beyond_32_bits():
    """Codes of more than 4 GB and values of more than 8 billion: the last rows are right."""
    rows, cols = 140000, 65536
    g = torch.Generator(device="cuda").manual_seed(1)
    codes = torch.randint(0, 256, (rows, cols // 2), dtype=torch.uint8, device="cuda", generator=g)
    scales = torch.randint(120, 124, (rows, cols // 32), dtype=torch.uint8, device="cuda", generator=g)
    tail = [0, rows - 3, rows - 2, rows - 1]
    c, s = codes[tail].contiguous(), scales[tail].contiguous()
    w = R.values(c.cpu().numpy(), s.cpu().numpy(), cols)
    for tokens in (1, 17, 40):
        for dtype in (torch.float16, torch.bfloat16):
            x = sample((tokens, cols), dtype, tokens, 2.0 ** -6)
            got = S.mx4_project(x, codes, scales, dtype=torch.float32)[:, tail]
            check_product(got, x, w, None, None, torch.float32)
    for tokens in (3, 130):
        xc, xs, x = packed((tokens, cols), tokens, 2.0 ** -6)
        check_matmul(S.mx4_matmul(xc, xs, codes, scales, dtype=torch.bfloat16)[:, tail], x, w, None, None, torch.bfloat16)
    values = S.mx4_dequantize(codes, scales, dtype=torch.bfloat16)
    assert torch.equal(values[tail].cpu().double(), torch.from_numpy(w))
    S.mx4_quantize_out(values, codes, scales)
    again = S.mx4_quantize(values[tail].contiguous())
    assert torch.equal(codes[tail], again[0]) and torch.equal(scales[tail], again[1])
    del codes, scales, values
    torch.cuda.empty_cache()
