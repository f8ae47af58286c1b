"""Attention over the paged 8-bit cache against a statement in 64 bits: element types, head layouts, lengths
from nothing to long contexts, windows, pages that end inside a tile, strides, garbage behind the contexts."""
from __future__ import annotations

import ctypes

import pytest
import torch

import decoder_reference as dr


@pytest.fixture(autouse=True)
def seeded():
    torch.manual_seed(1)


pytestmark = pytest.mark.gpu

SHAPES = [
    # lens [(rows, context)], heads, kv heads, dim, page
    ([(1, 1)], 1, 1, 64, 16),
    ([(1, 700)], 32, 8, 128, 64),
    ([(1, 33), (1, 1), (0, 5), (1, 64), (1, 257)], 8, 8, 64, 32),
    ([(4, 4), (2, 131), (3, 90)], 12, 4, 128, 16),
    ([(1, 0), (5, 3), (1, 17), (0, 0)], 6, 2, 128, 128),  # rows that see nothing, an empty cache
    ([(1, 9000), (1, 31)], 8, 1, 128, 128),
    ([(1, 20011)], 3, 1, 64, 16),
    ([(40, 77), (7, 7), (1, 300)], 7, 1, 64, 32),
    ([(130, 515), (64, 64)], 8, 2, 128, 64),
    ([(300, 300), (1, 50), (0, 3), (70, 1200), (129, 100)], 12, 4, 128, 16),  # the last: more rows than tokens
    ([(33, 3001)], 8, 1, 64, 128),
    ([(9, 5000), (16, 20)], 16, 2, 128, 32),
    ([(257, 257)], 5, 5, 64, 64),
    ([(3, 40), (2, 500)], 130, 1, 64, 16),
]


def run(pkg, lib, cache, q, n_heads, act, scale, window, out, workspace=None, max_q=None, max_ctx=None):
    ws = None if workspace is None else workspace.data_ptr()
    return lib.htp_b200_attn_paged(out.data_ptr(), out.stride(0), q.data_ptr(), q.stride(0), dr.ref(cache.desc()), n_heads,
                                   pkg.ACT_F32 if act == torch.float32 else pkg.ACT_F16, scale, window, max_q or cache.max_q,
                                   max_ctx or cache.max_ctx, ws, 0 if workspace is None else workspace.numel(), dr.stream())


def workspace_for(pkg, lib, cache, n_heads, act, max_q=None, max_ctx=None):
    n = lib.htp_b200_attn_workspace(dr.ref(cache.desc()), n_heads, pkg.ACT_F32 if act == torch.float32 else pkg.ACT_F16,
                                    max_q or cache.max_q, max_ctx or cache.max_ctx)
    assert n != ctypes.c_size_t(-1).value
    return torch.full((n,), 0xAB, dtype=torch.uint8, device="cuda") if n else None


@pytest.mark.parametrize("act", [torch.float32, torch.float16], ids=["f32", "f16"])
@pytest.mark.parametrize("kv", ["i8", "e4m3"])
@pytest.mark.parametrize("window", [0, 50])
@pytest.mark.parametrize("shape", range(len(SHAPES)))
def test_attention_matches_64_bits(pkg, lib, shape, window, kv, act):
    lens, heads, kv_heads, dim, page = SHAPES[shape]
    c = dr.Cache(pkg, lens, page=page, heads=kv_heads, dim=dim, kv=kv, seed=shape, extra_rows=3)
    c.spoil_behind([n for _, n in lens])
    wide = heads * dim
    buf = torch.randn((c.n_rows, wide + 32), device="cuda", generator=torch.Generator("cuda").manual_seed(7)).to(act)
    q = buf[:, 16:16 + wide]  # a band of a wider matrix
    out = torch.full((c.n_rows, wide + 64), 3.0, device="cuda", dtype=act)[:, 32:32 + wide]
    scale = 1.3 * dim ** -0.5
    assert run(pkg, lib, c, q, heads, act, scale, window, out, workspace_for(pkg, lib, c, heads, act)) == 0
    assert lib.htp_b200_stream_status(dr.stream()) == 0
    n = c.starts[-1]
    ref, mass, worst = dr.attention(c, q[:n], heads, scale, window)
    got = out[:n].double().view(n, heads, dim)
    bound = dr.attention_bound(ref, mass, worst, act == torch.float32, c.max_ctx)
    assert torch.isfinite(got).all()
    excess = ((got - ref).abs() / bound).max().item() if n else 0.0
    assert excess <= 1.0, excess
    assert (out[n:] == 3.0).all()  # rows behind the last sequence


@pytest.mark.parametrize("act", [torch.float32, torch.float16], ids=["f32", "f16"])
def test_workspace_changes_nothing_but_the_split(pkg, lib, act):
    """With no workspace and with one: both right; the same call twice: the same bits."""
    lens = [(1, 30000), (1, 12345)]
    c = dr.Cache(pkg, lens, page=64, heads=1, dim=128, kv="i8", seed=3)
    q = torch.randn((2, 4 * 128), device="cuda").to(act)
    ws = workspace_for(pkg, lib, c, 4, act)
    assert ws is not None
    outs = []
    for w in (ws, ws, None):
        out = torch.empty_like(q)
        assert run(pkg, lib, c, q, 4, act, 0.09, 0, out, w) == 0
        outs.append(out)
    assert torch.equal(outs[0], outs[1])
    ref, mass, worst = dr.attention(c, q, 4, 0.09, 0)
    bound = dr.attention_bound(ref, mass, worst, act == torch.float32, c.max_ctx)
    for out in outs:
        assert ((out.double().view(2, 4, 128) - ref).abs() <= bound).all()


@pytest.mark.parametrize("act", [torch.float32, torch.float16], ids=["f32", "f16"])
@pytest.mark.parametrize("rows", [1, 24])
@pytest.mark.parametrize("seed", [0, 11, 13, 38])  # (0, 11, 38: scores that jump from moderate to huge within a row)
def test_scales_far_apart_and_peaked_scores(pkg, lib, act, rows, seed):
    """Pages whose scales differ by many powers of two, scores up to some hundreds, large and tiny queries."""
    c = dr.Cache(pkg, [(rows, 400), (rows, 129)], page=16, heads=2, dim=64, kv="e4m3", seed=5, spread=4.0)
    c.scale["v"][0] = 2.0 ** -100  # (what the append gives a block of zeros)
    c.codes["v"][0] = 0
    q = torch.randn((2 * rows, 4 * 64), device="cuda", generator=torch.Generator("cuda").manual_seed(seed)) * (100.0 if act == torch.float16 else 1.0)
    if act == torch.float32:
        q[0] *= 3e5
        q[-1] *= 1e-6
    q = q.to(act)
    out = torch.empty_like(q)
    assert run(pkg, lib, c, q, 4, act, 0.125, 0, out) == 0
    ref, mass, worst = dr.attention(c, q, 4, 0.125, 0)
    bound = dr.attention_bound(ref, mass, worst, act == torch.float32, c.max_ctx)
    got = out.double().view_as(ref)
    if act == torch.float16:  # what lies above 65504 + 16 rounds to infinity: some of these values do
        got = torch.where(got.isinf() & (ref.abs() + bound >= 65520) & (got.sign() == ref.sign()), ref, got)
    assert ((got - ref).abs() <= bound).all()


def test_bad_entries_are_skipped_and_reported(pkg, lib):
    """A page number outside the cache, lengths over the bounds: no access, an error code, the others' rows right."""
    c = dr.Cache(pkg, [(1, 100), (1, 64), (2, 90)], page=32, heads=2, dim=128, kv="i8", seed=6)
    q = torch.randn((4, 4 * 128), device="cuda")
    ref, mass, worst = dr.attention(c, q, 4, 0.1, 0)
    bound = dr.attention_bound(ref, mass, worst, True, c.max_ctx)
    assert lib.htp_b200_stream_status(dr.stream()) == 0

    def rows_right(out, rows):
        return ((out.double().view_as(ref) - ref).abs() <= bound)[rows].all()

    good = c.table.clone()
    for bad in (-1, c.n_pages, 2 ** 31 - 1, -2 ** 31):
        c.table[0, 1] = bad
        out = torch.full_like(q, 3.0)
        assert run(pkg, lib, c, q, 4, torch.float32, 0.1, 0, out) == 0
        assert lib.htp_b200_stream_status(dr.stream()) == 301
        assert lib.htp_b200_stream_status(dr.stream()) == 0
        assert rows_right(out, [1, 2, 3])
    c.table.copy_(good)
    out = torch.full_like(q, 3.0)
    assert run(pkg, lib, c, q, 4, torch.float32, 0.1, 0, out, max_q=1) == 0  # the third sequence has two rows
    assert lib.htp_b200_stream_status(dr.stream()) == 302
    assert rows_right(out, [0, 1]) and (out[2:] == 3.0).all()
    for name, value, bad_rows in (("ctx_len", -5, [1]), ("ctx_len", 2 ** 31 - 1, [1]), ("q_start", 99, [0, 1])):
        t = getattr(c, name)
        keep = t.clone()
        t[1] = value
        out = torch.full_like(q, 3.0)
        assert run(pkg, lib, c, q, 4, torch.float32, 0.1, 0, out) == 0
        assert lib.htp_b200_stream_status(dr.stream()) == 302
        assert rows_right(out, [r for r in range(4) if r not in bad_rows]) and (out[bad_rows] == 3.0).all()
        t.copy_(keep)


def test_shared_pages_and_cache_past_4_gib(pkg, lib):
    """Two sequences that read the same pages; codes behind the 32-bit byte offsets."""
    c = dr.Cache(pkg, [(1, 200), (1, 150)], page=64, heads=2, dim=128, kv="i8", seed=8)
    c.table[1, :3] = c.table[0, :3]
    per_page = 2 * 64 * 128
    n_pages = (5 << 30) // per_page
    far = [n_pages - 1, n_pages - 7, 3, n_pages // 2 + 11]
    codes = {w: torch.empty((n_pages, 2, 64, 128), dtype=torch.uint8, device="cuda") for w in "kv"}
    scale = {w: torch.ones((n_pages, 2), device="cuda") for w in "kv"}
    for i in range(4):
        for w in "kv":
            codes[w][far[i]] = c.codes[w][c.table[0, i]]
            scale[w][far[i]] = c.scale[w][c.table[0, i]]
    q = torch.randn((2, 6 * 128), device="cuda")
    ref, mass, worst = dr.attention(c, q, 6, 0.1, 0)
    c.table[0, :4] = torch.tensor(far, device="cuda")
    c.table[1, :3] = c.table[0, :3]
    c.codes, c.scale, c.n_pages = codes, scale, n_pages
    out = torch.empty_like(q)
    assert run(pkg, lib, c, q, 6, torch.float32, 0.1, 0, out) == 0
    assert ((out.double().view_as(ref) - ref).abs() <= dr.attention_bound(ref, mass, worst, True, c.max_ctx)).all()


def test_captured_call_follows_the_lengths(pkg, lib):
    """A graph captured on a stream that the library has not seen, replayed after the lengths have changed."""
    c = dr.Cache(pkg, [(1, 500), (1, 90)], page=64, heads=2, dim=128, kv="e4m3", seed=9)
    q = torch.randn((2, 8 * 128), device="cuda").half()
    out = torch.empty_like(q)
    ws = workspace_for(pkg, lib, c, 8, q.dtype)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        assert run(pkg, lib, c, q, 8, q.dtype, 0.1, 0, out, ws) == 0
    for lens in ([(1, 500), (1, 90)], [(1, 77), (1, 320)], [(1, 1), (1, 0)]):
        c.lens = lens
        c.table[1, 2:6] = c.table[0, 2:6]
        c.ctx_len.copy_(torch.tensor([n for _, n in lens], dtype=torch.int32))
        q.normal_()
        out.fill_(3.0)
        graph.replay()
        torch.cuda.synchronize()
        ref, mass, worst = dr.attention(c, q, 8, 0.1, 0)
        assert ((out.double().view_as(ref) - ref).abs() <= dr.attention_bound(ref, mass, worst, False, c.max_ctx)).all()


@pytest.mark.parametrize("act", [torch.float32, torch.float16], ids=["f32", "f16"])
@pytest.mark.parametrize("rows", [1, 40])
def test_pages_behind_a_window_may_be_gone(pkg, lib, act, rows):
    """Entries of pages that no row sees any more name nothing; nothing is reported and the rows are right."""
    c = dr.Cache(pkg, [(rows, 700), (rows, 333)], page=16, heads=2, dim=64, kv="e4m3", seed=10)
    q = torch.randn((2 * rows, 8 * 64), device="cuda").to(act)
    ref, mass, worst = dr.attention(c, q, 8, 0.125, 50)
    for b, (r, n) in enumerate(c.lens):
        c.table[b, :(n - r + 1 - 50) // 16] = -7
    out = torch.empty_like(q)
    assert run(pkg, lib, c, q, 8, act, 0.125, 50, out) == 0
    assert lib.htp_b200_stream_status(dr.stream()) == 0
    assert ((out.double().view_as(ref) - ref).abs() <= dr.attention_bound(ref, mass, worst, act == torch.float32, c.max_ctx)).all()


@pytest.mark.parametrize("act", [torch.float32, torch.float16], ids=["f32", "f16"])
@pytest.mark.parametrize("rows", [2, 40])
def test_rows_do_not_see_each_other(pkg, lib, act, rows):
    """NaN and infinities in some rows' queries leave the other rows as they are; a scale of 0 over codes of 0."""
    c = dr.Cache(pkg, [(rows, 300), (rows, rows)], page=32, heads=2, dim=128, kv="i8", seed=11)
    c.codes["v"][c.table[0, 2]], c.scale["v"][c.table[0, 2]] = 0, 0.0
    c.codes["k"][c.table[0, 3]], c.scale["k"][c.table[0, 3]] = 0, 0.0
    q = torch.randn((2 * rows, 6 * 128), device="cuda").to(act)
    ref, mass, worst = dr.attention(c, q, 6, 0.1, 0)
    q[1, 5] = float("nan")  # head 0
    q[rows, 200] = float("inf")  # head 1
    out = torch.empty_like(q)
    assert run(pkg, lib, c, q, 6, act, 0.1, 0, out) == 0
    got = out.double().view_as(ref)
    keep = torch.ones_like(ref, dtype=torch.bool)
    keep[1, 0] = keep[rows, 1] = False
    bound = dr.attention_bound(ref, mass, worst, act == torch.float32, c.max_ctx)
    assert ((got - ref).abs() <= bound)[keep].all()
    assert torch.isnan(got[1, 0]).all()


def test_bounds_of_a_call_above_what_it_has(pkg, lib):
    """max_q and max_ctx as a captured program would give them, far above this step's rows and contexts."""
    c = dr.Cache(pkg, [(1, 30), (3, 200), (1, 5)], page=16, heads=2, dim=64, kv="i8", seed=12, table_pad=600, extra_rows=60)
    q = torch.randn((65, 4 * 64), device="cuda")
    ref, mass, worst = dr.attention(c, q[:5], 4, 0.125, 0)
    bound = dr.attention_bound(ref, mass, worst, True, c.max_ctx)
    for max_q, max_ctx in ((3, 200), (3, 9000), (8, 9000), (64, 200), (64, 9000)):
        ws = workspace_for(pkg, lib, c, 4, q.dtype, max_q, max_ctx)
        for w in (ws, None):
            out = torch.full_like(q, 3.0)
            assert run(pkg, lib, c, q, 4, q.dtype, 0.125, 0, out, w, max_q, max_ctx) == 0
            assert ((out[:5].double().view_as(ref) - ref).abs() <= bound).all() and (out[5:] == 3.0).all()
    assert lib.htp_b200_stream_status(dr.stream()) == 0


def test_calls_on_two_streams_at_once(pkg, lib):
    """The same cache read by two streams, each with its own output and workspace, again and again."""
    c = dr.Cache(pkg, [(1, 30000), (1, 700)], page=64, heads=1, dim=128, kv="e4m3", seed=13)
    streams = [torch.cuda.Stream() for _ in range(2)]
    qs = [torch.randn((2, 4 * 128), device="cuda").half() for _ in streams]
    outs, wss = [torch.empty_like(q) for q in qs], [workspace_for(pkg, lib, c, 4, torch.float16) for _ in streams]
    torch.cuda.synchronize()
    for _ in range(20):
        for s, q, out, ws in zip(streams, qs, outs, wss):
            with torch.cuda.stream(s):
                assert run(pkg, lib, c, q, 4, q.dtype, 0.1, 0, out, ws) == 0
    torch.cuda.synchronize()
    for q, out in zip(qs, outs):
        ref, mass, worst = dr.attention(c, q, 4, 0.1, 0)
        assert ((out.double().view_as(ref) - ref).abs() <= dr.attention_bound(ref, mass, worst, False, c.max_ctx)).all()


@pytest.mark.parametrize("heads", [2, 20])  # (the kernels for few and for many rows of a key/value head)
def test_hundreds_of_sequences(pkg, lib, heads):
    """More sequences than a CTA has threads, some of no rows, some of no tokens."""
    c = dr.Cache(pkg, [(i % 3, i % 3 + (i * 7) % 50) for i in range(700)], page=16, heads=1, dim=64, kv="i8", seed=14, extra_rows=5)
    n = c.starts[-1]
    q = torch.randn((c.n_rows, heads * 64), device="cuda")
    out = torch.full_like(q, 3.0)
    assert run(pkg, lib, c, q, heads, torch.float32, 0.125, 0, out) == 0
    assert lib.htp_b200_stream_status(dr.stream()) == 0
    ref, mass, worst = dr.attention(c, q[:n], heads, 0.125, 0)
    assert ((out[:n].double().view_as(ref) - ref).abs() <= dr.attention_bound(ref, mass, worst, True, c.max_ctx)).all()
    assert (out[n:] == 3.0).all()
