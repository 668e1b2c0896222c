"""bfloat16 products of few rows whose operands do not start on 16 bytes: the weight-streaming kernel, which loads 16 bytes at a time, does
not take them, whatever their strides; the library does."""

import pytest
import torch

from tinyvllm_b200.ops import gemm, kernels

BF16 = torch.bfloat16


def placed(rows, columns, offset, stride, device="cpu", values=None):
    """[rows, columns] that begins ``offset`` elements into a buffer, with rows ``stride`` apart."""
    buffer = torch.zeros(offset + rows * stride + 8, dtype=BF16, device=device)
    view = buffer[offset:offset + rows * stride].view(rows, stride)[:, :columns]
    return view if values is None else view.copy_(values)


@pytest.mark.parametrize("offset", [0, 1, 4, 7, 8])
@pytest.mark.parametrize("which", ["x", "weight"])
def test_which_kernel_takes_them(which, offset):
    operands = dict(x=placed(3, 16, 0, 24), weight=placed(24, 16, 0, 16))
    operands[which] = placed(operands[which].shape[0], 16, offset, 24)
    assert operands[which].stride() == (24, 1)
    assert gemm.small(**operands) == (offset % 8 == 0)


@pytest.mark.parametrize("which", ["x", "w", "residual"])
def test_the_kernels_face_refuses_them(which, monkeypatch):
    monkeypatch.setattr(kernels, "_need_cuda", lambda *tensors: None)
    operands = dict(x=placed(3, 16, 0, 16), w=placed(24, 16, 0, 16), residual=placed(3, 16, 0, 16))
    operands[which] = placed(operands[which].shape[0], 16, 4, 16)
    assert operands[which].is_contiguous()
    with pytest.raises(kernels.KernelError, match="16 bytes"):
        kernels.gemm_small_m(operands.pop("x"), operands.pop("w"), norm_weight=torch.ones(16, dtype=BF16), **operands)


@pytest.mark.gpu
@pytest.mark.parametrize("offset", [1, 2, 4, 7, 8])
@pytest.mark.parametrize("k, n", [(8, 872), (64, 40), (1024, 136)])
@pytest.mark.parametrize("m", [1, 7, 14, 16, 17])
def test_products_and_adapters(m, k, n, offset):
    from test_adapters_gpu import adapted, check, made
    from tinyvllm_b200.ops import linear

    for which in ("x", "weight"):
        s = made(m, k, n, 8, 3)
        s[which] = placed(s[which].shape[0], k, offset, k + 8, "cuda", s[which])
        x, w = s["x"].double(), s["weight"].double()
        sizes, want = x.abs() @ w.abs().t(), x @ w.t()
        # float32 results: sums of k products, 2^-23 of their sizes a step, and a rounding
        bound = (k + 8) * 2.0**-23 * sizes
        got = linear(s["x"], s["weight"], out_dtype=torch.float32)
        assert ((got.double() - want).abs() <= bound + 2.0**-24 * want.abs()).all()
        check(adapted(**s, out_dtype=torch.float32), s)
        # bfloat16 results: the library may round pieces of such a sum, none larger than the sizes; four roundings are allowed
        base = linear(s["x"], s["weight"])
        assert ((base.double() - want).abs() <= bound + 4 * 2.0**-8 * sizes).all()
        got = adapted(**s)
        extra = torch.zeros_like(want)                     # the adapters' part, on the projection as it is
        extra_sizes = torch.zeros_like(want)
        for a in range(3):
            rows = (s["ids"] == a).nonzero()[:, 0]
            down, up, scale = s["down"][a].double(), s["up"][a].double(), s["scales"][a].double()
            extra[rows] = scale * (x[rows] @ down.t()) @ up.t()
            extra_sizes[rows] = scale.abs() * (x[rows].abs() @ down.abs().t()) @ up.abs().t()
        total = base.double() + extra
        bound = ((k + 24) * 2.0**-23 + 2.0**-16) * extra_sizes + 2.0**-23 * total.abs()
        assert ((got.double() - total).abs() <= bound + 2.0**-8 * (total.abs() + bound)).all()
        assert torch.equal(got[s["ids"] < 0], base[s["ids"] < 0])
