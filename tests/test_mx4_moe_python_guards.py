"""Refusals of the Python calls, without a GPU: tensors that say they are on one. A call that is not
refused would come to the library (or to a missing driver) with another error."""
import pytest
import torch

import swiglu_b200 as S


class Claimed(torch.Tensor):
    is_cuda = True


def t(*shape, dtype=torch.float16, grad=False):
    return torch.zeros(*shape, dtype=dtype).as_subclass(Claimed).requires_grad_(grad)


def u8(*shape):
    return t(*shape, dtype=torch.uint8)


def refused(fn, *args, match, **kw):
    with pytest.raises(RuntimeError, match=match):
        fn(*args, **kw)


def test_no_tensor_may_require_gradients():
    """The outputs neither: a leaf would be written in silence."""
    m = "disable gradients"
    x, q, s = t(2, 64), u8(8, 32), u8(8, 2)
    refused(S.mx4_quantize_out, t(2, 64, grad=True), u8(2, 32), u8(2, 2), match=m)
    for dtype in (torch.float16, torch.bfloat16, torch.float32):
        refused(S.mx4_dequantize_out, q, s, t(8, 64, dtype=dtype, grad=True), match=m)
    for dtype in (torch.float16, torch.float32):
        refused(S.mx4_project_out, x, q, s, t(2, 8, dtype=dtype, grad=True), match=m)
    refused(S.mx4_project_out, t(2, 64, grad=True), q, s, t(2, 8), match=m)
    refused(S.mx4_project_out, x, q, s, t(2, 8), t(8, grad=True), match=m)
    refused(S.mx4_project_out, x, q, s, t(2, 8), None, t(2, 8, grad=True), match=m)
    refused(S.mx4_matmul_out, u8(2, 32), u8(2, 2), q, s, t(2, 8, grad=True), match=m)
    refused(S.mx4_matmul_out, u8(2, 32), u8(2, 2), q, s, t(2, 8), t(8, grad=True), match=m)
    for i in range(7):
        a = [t(2, 64, grad=i == 0), t(4, 64, grad=i == 1), t(4, 32, 64, grad=i == 2), t(4, 32, 64, grad=i == 3),
             t(4, 64, 32, grad=i == 4), t(2, 64, grad=i == 5)]
        refused(S.moe_out, *a, u8(1 << 20), 2, weights=t(2, 2, dtype=torch.float32, grad=i == 6), match=m)


def test_sizes_beyond_32_bits_are_refused():
    """Not cut to their low bits: 2^32 + 2 places are not two."""
    big = 1 << 32
    for sizes in ((1 + big, 8, 2, 64), (1, 8 + big, 2, 64), (1, 8, 2 + big, 64), (1, 8, 2, 64 + big),
                  (1 - big, 8, 2, 64), (1, 8, 2 - big, 64)):
        refused(S.moe_workspace, *sizes, device="cpu", match="invalid shape")
    a = [t(2, 64), t(4, 64), t(4, 32, 64), t(4, 32, 64), t(4, 64, 32), t(2, 64), u8(1 << 20)]
    for topk in (2 + big, 2 - big, 0, 5, 17):
        refused(S.moe_out, *a, topk, match="invalid shape")
    refused(S.moe, *a[:5], 2 + big, match="invalid shape")
