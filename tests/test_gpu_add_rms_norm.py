"""Residual and norms between two blocks against a statement in 64 bits."""
from __future__ import annotations

import pytest
import torch

import decoder_reference as dr

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def seeded():
    torch.manual_seed(1)


def statement(x, block, post, gate, weight, block_scale, eps):
    h = x.double()
    if block is not None:
        b = block.double()
        if post is not None:
            b = b / (b.square().mean(1, keepdim=True) + eps).sqrt() * post.double()
        if gate is not None:
            b = b * gate.double()
        h = h + block_scale * b
    n = h / (h.square().mean(1, keepdim=True) + eps).sqrt()
    return h, n if weight is None else n * weight.double()


def call(pkg, lib, h, out, x, block, post, gate, gate_stride, weight, block_scale, eps, n=None):
    p = lambda t: None if t is None else t.data_ptr()  # noqa: E731
    f16 = out is not None and out.dtype == torch.float16
    return lib.htp_b200_add_rms_norm(p(h), p(out), p(x), p(block), p(post), p(gate), gate_stride, p(weight), block_scale, eps,
                                     n or x.shape[1], x.shape[0], pkg.ACT_F16 if f16 else pkg.ACT_F32, dr.stream())


def check(h, out, x, want_h, want_n, block_part):
    # fp32: the post norm's factor is off by less than (n + 8) / 2 roundings that partly cancel - taken as 16 roundings
    # of the block's part (pairwise sums of at most 64 terms in a row), the sum by one of its largest term; the norm likewise
    e = 2.0 ** -24
    if h is not None:
        assert ((h.double() - want_h).abs() <= 16 * e * block_part + 2 * e * (x.double().abs() + block_part)).all()
    if out is not None:
        rms = want_n.square().mean(1, keepdim=True).sqrt()
        slack = 32 * e * (want_n.abs() + rms * (block_part + x.double().abs()) / (want_h.abs() + 1e-30).clamp(min=want_h.square().mean(1, keepdim=True).sqrt()))
        if out.dtype == torch.float16:
            slack = slack + 2.0 ** -11 * want_n.abs() + 2.0 ** -25
        assert ((out.double() - want_n).abs() <= slack).all(), ((out.double() - want_n).abs() / slack).max()


@pytest.mark.parametrize("out_type", [torch.float32, torch.float16], ids=["f32", "f16"])
@pytest.mark.parametrize("post,gate", [(False, None), (True, None), (True, "row"), (False, "all")])
@pytest.mark.parametrize("rows,n", [(1, 1), (3, 32), (2, 100), (5, 4096), (7, 4097), (2, 8192), (3, 16384), (2, 20001), (2, 40000), (300, 257)])
def test_matches_64_bits(pkg, lib, rows, n, post, gate, out_type):
    g = torch.Generator("cuda").manual_seed(n)
    x, block = (torch.randn((rows, n), generator=g, device="cuda") * s for s in (3.0, 0.5))
    weight, pw = (1 + 0.2 * torch.randn(n, generator=g, device="cuda") for _ in range(2))
    pw = pw if post else None
    gv = None if gate is None else torch.randn((rows if gate == "all" else 1, n), generator=g, device="cuda")
    h, out = torch.empty_like(x), torch.empty((rows, n), device="cuda", dtype=out_type)
    assert call(pkg, lib, h, out, x, block, pw, gv, n if gate == "all" else 0, weight, 0.7, 1e-5) == 0
    want_h, want_n = statement(x, block, pw, gv, weight, float(torch.tensor(0.7)), float(torch.tensor(1e-5)))
    check(h, out, x, want_h, want_n * 1.0, (want_h - x.double()).abs())


def test_optional_parts_and_in_place(pkg, lib):
    g = torch.Generator("cuda").manual_seed(1)
    x, block = (torch.randn((4, 4096), generator=g, device="cuda") for _ in range(2))
    want_h, want_n = statement(x, block, None, None, None, 1.0, 1e-6)
    zero = torch.zeros_like(want_h)
    out = torch.empty_like(x)
    assert call(pkg, lib, None, out, x, block, None, None, 0, None, 1.0, 1e-6) == 0
    check(None, out, x, want_h, want_n, block.double().abs())
    h = torch.empty_like(x)
    assert call(pkg, lib, h, None, x, block, None, None, 0, None, 1.0, 1e-6) == 0
    check(h, None, x, want_h, want_n, block.double().abs())
    assert call(pkg, lib, None, out, x, None, None, None, 0, None, 1.0, 1e-6) == 0  # a first block's input norm
    check(None, out, x, *statement(x, None, None, None, None, 1.0, 1e-6), zero)
    for n in (4096, 40000):  # h over x, norm over block
        x, block = (torch.randn((3, n), generator=g, device="cuda") for _ in range(2))
        want_h, want_n = statement(x, block, None, None, None, 1.0, 1e-6)
        x1, b1 = x.clone(), block.clone()
        assert call(pkg, lib, x1, b1, x1, b1, None, None, 0, None, 1.0, 1e-6) == 0
        check(x1, b1, x, want_h, want_n, block.double().abs())
        x1 = x.clone()
        assert call(pkg, lib, None, x1, x1, block, None, None, 0, None, 1.0, 1e-6) == 0  # norm over x
        check(None, x1, x, want_h, want_n, block.double().abs())


def test_a_row_of_zeros_no_numbers_and_other_rows(pkg, lib):
    x, block = torch.randn((4, 512), device="cuda"), torch.randn((4, 512), device="cuda")
    x[1], block[1] = 0, 0
    x[2, 7] = float("nan")
    h, out = torch.empty_like(x), torch.empty_like(x)
    assert call(pkg, lib, h, out, x, block, torch.ones(512, device="cuda"), None, 0, None, 1.0, 1e-5) == 0
    assert (h[1] == 0).all() and (out[1] == 0).all()
    assert torch.isnan(out[2]).all() and torch.isnan(h[2]).sum() == 1
    assert torch.isfinite(out[[0, 3]]).all()
    # operands at any alignment of their type
    big = torch.randn(4 * 512 + 1, device="cuda")
    xs = big[1:].view(4, 512)
    out2 = torch.empty_like(x)
    assert call(pkg, lib, None, out2, xs, None, None, None, 0, None, 1.0, 1e-5) == 0
    want_h, want_n = statement(xs, None, None, None, None, 1.0, 1e-5)
    check(None, out2, xs, want_h, want_n, torch.zeros_like(want_h))
