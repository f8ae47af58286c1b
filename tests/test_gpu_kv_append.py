"""Append to the paged 8-bit cache: bytes and scales against the definition's fp32 steps, and against the rotation in 64 bits."""
from __future__ import annotations

import pytest
import torch

import decoder_reference as dr

pytestmark = pytest.mark.gpu

LENS = [
    [(1, 1)],
    [(1, 701), (1, 64), (1, 65), (0, 9), (1, 128)],
    [(5, 5), (130, 300), (64, 64), (1, 17), (33, 63)],
]


def call(pkg, lib, c, k, v, q, q_out, heads, rope, act=None):
    code = {torch.float32: pkg.ACT_F32, torch.float16: pkg.ACT_F16}
    return lib.htp_b200_kv_append(dr.ref(c.desc()), None if rope is None else dr.ref(rope), k.data_ptr(), k.stride(0), v.data_ptr(),
                                  v.stride(0), None if q is None else q.data_ptr(), 0 if q is None else q.stride(0),
                                  None if q is None else q_out.data_ptr(), 0 if q is None else q_out.stride(0), heads, code[k.dtype],
                                  pkg.ACT_F32 if q is None else code[q_out.dtype], dr.stream())


def angles(n, rot):
    a = torch.arange(n, dtype=torch.float64, device="cuda")[:, None] * 10000.0 ** (-torch.arange(0, rot, 2, dtype=torch.float64, device="cuda") / rot)
    return torch.cat([a.cos(), a.sin()], 1).float().contiguous()


def inputs(c, heads, act, seed):
    g = torch.Generator("cuda").manual_seed(seed)
    x = torch.randn((c.n_rows, (heads + 2 * c.heads) * c.dim), generator=g, device="cuda") * torch.exp(torch.randn((c.n_rows, 1), generator=g, device="cuda"))
    return x.to(act).split([heads * c.dim, c.heads * c.dim, c.heads * c.dim], 1)


def same_cache(c, want):
    for w in "kv":
        assert torch.equal(c.scale[w], want[w][1])
        a, b = dr.decode(c.codes[w], c.kv), dr.decode(want[w][0], c.kv)
        assert torch.equal(a.nan_to_num(1e9), b.nan_to_num(1e9)), (a != b).sum()


@pytest.mark.parametrize("act", [torch.float32, torch.float16], ids=["f32", "f16"])
@pytest.mark.parametrize("kv", ["i8", "e4m3"])
@pytest.mark.parametrize("mode,rot", [(0, 8), (1, 64), (2, 64), (2, 24), (1, 8)])
@pytest.mark.parametrize("page,dim", [(16, 64), (32, 128), (64, 64), (128, 128)])
@pytest.mark.parametrize("lens", range(len(LENS)))
def test_append_matches_its_definition(pkg, lib, lens, page, dim, mode, rot, kv, act):
    heads = 6
    c = dr.Cache(pkg, LENS[lens], page=page, heads=2, dim=dim, kv=kv, seed=lens, extra_rows=2, spread=2.0)
    c.spoil_behind([n - q for q, n in c.lens])
    q, k, v = inputs(c, heads, act, 3 + lens)
    table = angles(c.max_ctx, rot)
    rope = pkg.Rope(table=table.data_ptr(), positions=None, table_len=len(table), rot_dim=rot, mode=mode)
    want = dr.append(c, k, v, table, rot, mode)
    q_out = torch.full((c.n_rows, heads * dim + 8), 3.0, device="cuda")[:, 8:]
    assert call(pkg, lib, c, k, v, q, q_out, heads, rope) == 0
    assert lib.htp_b200_stream_status(dr.stream()) == 0
    same_cache(c, want)
    n = c.starts[-1]
    pos = torch.cat([torch.arange(t - r, t, device="cuda") for r, t in c.lens])
    x = q[:n].float().reshape(n, heads, dim)
    assert torch.equal(q_out[:n].reshape(n, heads, dim), dr.rotate(x, table[pos], rot, mode))
    if mode:  # and the rotation itself, in 64 bits: two products and a sum, each rounded once
        ref = dr.rotate(x.double(), table[pos].double(), rot, mode)
        size = dr.rotate(x.double().abs(), torch.cat([table[pos][:, :rot // 2].double().abs(), -table[pos][:, rot // 2:].double().abs()], 1), rot, mode).abs()
        pair = size.amax(2, keepdim=True) + x.double().abs().amax(2, keepdim=True)
        assert ((q_out[:n].reshape(n, heads, dim).double() - ref).abs() <= 2.0 ** -22 * pair).all()
    assert (q_out[n:] == 3.0).all()
    # the same rows again change nothing
    assert call(pkg, lib, c, k, v, q, q_out, heads, rope) == 0
    same_cache(c, want)


@pytest.mark.parametrize("kv", ["i8", "e4m3"])
def test_token_by_token_growth(pkg, lib, kv):
    """A page filled one token at a time, each larger than all before: older codes follow the scale at every step."""
    c = dr.Cache(pkg, [(1, 40), (1, 80)], page=32, heads=2, dim=64, kv=kv, seed=2)
    for step in range(1, 41):
        c.lens = [(1, step), (1, 40 + step)]
        c.ctx_len.copy_(torch.tensor([n for _, n in c.lens], dtype=torch.int32))
        _, k, v = inputs(c, 2, torch.float32, step)
        k, v = k * 1.2 ** step, v * (0.0 if step % 7 == 0 else 1.0)
        want = dr.append(c, k, v, None, 0, 0)
        assert call(pkg, lib, c, k, v, None, None, 0, None) == 0
        same_cache(c, want)


@pytest.mark.parametrize("kv", ["i8", "e4m3"])
def test_no_numbers_infinities_zeros_and_extremes(pkg, lib, kv):
    c = dr.Cache(pkg, [(20, 20), (3, 36)], page=16, heads=2, dim=64, kv=kv, seed=4)
    _, k, v = (t.clone() for t in inputs(c, 2, torch.float32, 9))
    k[0, 5], k[1, 6], k[2, 7] = float("nan"), float("inf"), -float("inf")
    v[16:20] = 0.0
    k[16:20] = 1e-38
    v[20, 3], v[21, 3] = 3e38, -3e38
    k[20:23, 64:] = float("nan")
    want = dr.append(c, k, v, None, 0, 0)
    assert call(pkg, lib, c, k, v, None, None, 0, None) == 0
    same_cache(c, want)


def test_positions_in_place_and_fp16_queries(pkg, lib):
    c = dr.Cache(pkg, [(3, 50), (2, 2)], page=16, heads=1, dim=128, kv="i8", seed=5, extra_rows=1)
    pos = torch.tensor([7, 0, 99, 3, 3, -77], dtype=torch.int32, device="cuda")  # (the last row is nobody's)
    table = angles(100, 128)
    rope = pkg.Rope(table=table.data_ptr(), positions=pos.data_ptr(), table_len=100, rot_dim=128, mode=2)
    q, k, v = (t.contiguous() for t in inputs(c, 4, torch.float32, 5))
    want = dr.append(c, k, v, table, 128, 2, pos)
    out16 = torch.empty((6, 512), dtype=torch.float16, device="cuda")
    assert call(pkg, lib, c, k, v, q, out16, 4, rope) == 0
    same_cache(c, want)
    ref = dr.rotate(q[:5].view(5, 4, 128), table[pos[:5].long()], 128, 2).reshape(5, 512)
    assert torch.equal(out16[:5], ref.half())
    last = q[5].clone()
    assert call(pkg, lib, c, k, v, q, q, 4, rope) == 0  # in place
    assert torch.equal(q[:5], ref) and torch.equal(q[5], last)
    assert lib.htp_b200_stream_status(dr.stream()) == 0


def test_bad_entries_are_skipped_and_reported(pkg, lib):
    c = dr.Cache(pkg, [(3, 40), (2, 20)], page=16, heads=2, dim=64, kv="i8", seed=6, table_pad=0)
    _, k, v = inputs(c, 2, torch.float32, 2)
    table = angles(64, 64)
    assert lib.htp_b200_stream_status(dr.stream()) == 0
    want = dr.append(c, k, v, table, 64, 1)

    def attempt(code, first_unchanged, **rope_args):
        before = {w: (c.codes[w].clone(), c.scale[w].clone()) for w in "kv"}
        args = dict(table=table.data_ptr(), positions=None, table_len=64, rot_dim=64, mode=1)
        args.update(rope_args)
        assert call(pkg, lib, c, k, v, None, None, 0, pkg.Rope(**args)) == 0
        assert lib.htp_b200_stream_status(dr.stream()) == code
        page = int(keep[0, 2])
        if first_unchanged:
            assert torch.equal(c.codes["k"][page], before["k"][0][page]) and torch.equal(c.scale["k"][page], before["k"][1][page])
        assert torch.equal(c.codes["k"][int(keep[1, 1])], want["k"][0][int(keep[1, 1])])

    keep = c.table.clone()
    for bad in (-1, c.n_pages, 2 ** 31 - 1):
        c.table[0, 2] = bad
        attempt(301, True)
    c.table.copy_(keep)
    attempt(303, True, table_len=39)  # position 39 lies behind it
    for value in (-1, 2, 49, 2 ** 31 - 1):  # no context of 3 rows in a table of three pages
        c.ctx_len[0] = value
        attempt(302, True)
    c.ctx_len[0] = 40
    attempt(0, False)
    same_cache(c, want)


def test_hundreds_of_sequences(pkg, lib):
    """More sequences than a CTA has threads, some of no rows."""
    c = dr.Cache(pkg, [(i % 4, i % 4 + (i * 7) % 40) for i in range(600)], page=16, heads=1, dim=64, kv="e4m3", seed=7, extra_rows=3)
    q, k, v = inputs(c, 2, torch.float32, 8)
    table = angles(c.max_ctx, 32)
    rope = pkg.Rope(table=table.data_ptr(), positions=None, table_len=len(table), rot_dim=32, mode=1)
    want = dr.append(c, k, v, table, 32, 1)
    q_out = torch.full((c.n_rows, 128), 3.0, device="cuda")
    assert call(pkg, lib, c, k, v, q, q_out, 2, rope) == 0
    assert lib.htp_b200_stream_status(dr.stream()) == 0
    same_cache(c, want)
    n = c.starts[-1]
    pos = torch.cat([torch.arange(t - r, t, device="cuda") for r, t in c.lens])
    assert torch.equal(q_out[:n].reshape(n, 2, 64), dr.rotate(q[:n].float().reshape(n, 2, 64), table[pos], 32, 1))
    assert (q_out[n:] == 3.0).all()
