"""Refusals of the operators around a decoder's matmuls: decided on the host, before any launch, with and
without a GPU (addresses below are never followed)."""
from __future__ import annotations

import ctypes

import pytest

A = 1 << 20  # an aligned address that nothing follows


def kv(pkg, **change):
    f = dict(k_codes=A, v_codes=2 * A, k_scale=3 * A, v_scale=4 * A, page_table=5 * A, q_start=6 * A, ctx_len=7 * A, n_pages=10, page_size=16, n_kv_heads=2,
             head_dim=64, kv_type=pkg.KV_I8, n_seqs=2, table_stride=4, n_rows=5)
    f.update(change)
    return ctypes.byref(pkg.PagedKv(**f))


BAD_CACHES = [dict(k_codes=None), dict(v_codes=None), dict(k_scale=None), dict(v_scale=None), dict(page_table=None), dict(q_start=None), dict(ctx_len=None),
              dict(k_codes=A + 8), dict(v_codes=A + 1), dict(k_scale=A + 2), dict(page_table=A + 1), dict(n_pages=0), dict(n_pages=-1), dict(page_size=0), dict(page_size=8),
              dict(page_size=48), dict(page_size=256), dict(n_kv_heads=0), dict(head_dim=0), dict(head_dim=96), dict(head_dim=256), dict(kv_type=2), dict(kv_type=-1),
              dict(n_seqs=0), dict(table_stride=0), dict(n_rows=0), dict(n_rows=-3)]


def append(pkg, lib, cache=None, rope=None, k=8 * A, ks=128, v=9 * A, vs=128, q=10 * A, qs=256, qo=11 * A, qos=256, heads=4, act=0, qt=0):
    return lib.htp_b200_kv_append(cache or kv(pkg), rope, k, ks, v, vs, q, qs, qo, qos, heads, act, qt, None)


def attn(pkg, lib, cache=None, out=10 * A, os=256, q=11 * A, qs=256, heads=4, act=0, scale=0.1, window=0, max_q=2, max_ctx=64, ws=None, wsb=0):
    return lib.htp_b200_attn_paged(out, os, q, qs, cache or kv(pkg), heads, act, scale, window, max_q, max_ctx, ws, wsb, None)


@pytest.mark.parametrize("change", BAD_CACHES, ids=str)
def test_bad_caches(pkg, lib, change):
    assert append(pkg, lib, kv(pkg, **change)) == -1
    assert attn(pkg, lib, kv(pkg, **change)) == -1


def test_null_cache(pkg, lib):
    assert lib.htp_b200_kv_append(None, None, 8 * A, 128, 9 * A, 128, None, 0, None, 0, 0, 0, 0, None) == -1
    assert lib.htp_b200_attn_paged(10 * A, 256, 11 * A, 256, None, 4, 0, 0.1, 0, 1, 1, None, 0, None) == -1


@pytest.mark.parametrize("change", [dict(k=None), dict(v=None), dict(k=8 * A + 4), dict(ks=127), dict(ks=130), dict(ks=64), dict(vs=0), dict(vs=-128), dict(qs=255),
                                    dict(qo=None), dict(qo=11 * A + 8), dict(qos=128), dict(heads=0), dict(heads=-1), dict(act=2), dict(act=-1), dict(qt=7),
                                    dict(act=1, ks=132), dict(qo=10 * A, qt=1), dict(qo=10 * A, qos=512), dict(qo=10 * A + 1024), dict(qo=A), dict(qo=8 * A), dict(qo=9 * A)], ids=str)
def test_bad_appends(pkg, lib, change):
    assert append(pkg, lib, **change) == -1


def test_appends_into_overlapping_arrays(pkg, lib):
    assert append(pkg, lib, kv(pkg, v_codes=A + 16)) == -1 and append(pkg, lib, kv(pkg, v_scale=3 * A)) == -1
    assert append(pkg, lib, k=A) == -1 and append(pkg, lib, v=2 * A + 1024) == -1


@pytest.mark.parametrize("change", [dict(table=None), dict(table=A + 4), dict(table_len=0), dict(rot_dim=0), dict(rot_dim=12), dict(rot_dim=72), dict(mode=3), dict(mode=-1),
                                    dict(positions=A + 2)], ids=str)
def test_bad_rotations(pkg, lib, change):
    f = dict(table=12 * A, positions=None, table_len=9, rot_dim=64, mode=pkg.ROPE_PAIRS)
    f.update(change)
    assert append(pkg, lib, rope=ctypes.byref(pkg.Rope(**f))) == -1


@pytest.mark.parametrize("change", [dict(out=None), dict(q=None), dict(out=10 * A + 4), dict(q=11 * A + 8), dict(os=255), dict(qs=250), dict(heads=0), dict(heads=3), dict(act=5),
                                    dict(scale=0.0), dict(scale=-1.0), dict(scale=float("nan")), dict(scale=float("inf")), dict(window=-1), dict(max_q=0), dict(max_q=6),
                                    dict(max_ctx=0), dict(max_ctx=65), dict(ws=A + 8, wsb=64), dict(out=11 * A), dict(out=A), dict(ws=10 * A, wsb=64)], ids=str)
def test_bad_attention(pkg, lib, change):
    assert attn(pkg, lib, **change) == -1


def test_workspace_is_host_arithmetic(pkg, lib):
    bad = ctypes.c_size_t(-1).value
    assert lib.htp_b200_attn_workspace(None, 4, 0, 1, 1) == bad
    assert lib.htp_b200_attn_workspace(kv(pkg), 3, 0, 1, 1) == bad
    assert lib.htp_b200_attn_workspace(kv(pkg), 4, 0, 1, 65) == bad
    no_pointers = dict(k_codes=None, v_codes=None, k_scale=None, v_scale=None, page_table=None, q_start=None, ctx_len=None)
    assert lib.htp_b200_attn_workspace(kv(pkg, **no_pointers), 4, 0, 1, 64) == 0
    long = dict(no_pointers, table_stride=10000, n_seqs=1)
    assert 0 < lib.htp_b200_attn_workspace(kv(pkg, **long), 4, 0, 1, 160000) < 1 << 20


def norm(lib, h=A, out=2 * A, x=3 * A, block=4 * A, post=5 * A, gate=6 * A, gs=64, w=7 * A, bs=1.0, eps=1e-5, n=64, rows=2, t=0):
    return lib.htp_b200_add_rms_norm(h, out, x, block, post, gate, gs, w, bs, eps, n, rows, t, None)


@pytest.mark.parametrize("change", [dict(x=None), dict(h=None, out=None), dict(n=0), dict(n=-4), dict(rows=0), dict(t=2), dict(eps=-1.0), dict(eps=float("nan")),
                                    dict(bs=float("inf")), dict(block=None), dict(block=None, post=None), dict(block=None, gate=None), dict(gs=63), dict(gs=-64), dict(x=3 * A + 2),
                                    dict(out=2 * A + 1, t=1), dict(h=3 * A + 4), dict(out=3 * A + 64), dict(out=3 * A, t=1), dict(out=A), dict(h=6 * A), dict(out=7 * A),
                                    dict(h=5 * A)], ids=str)
def test_bad_norms(lib, change):
    assert norm(lib, **change) == -1


GOOD = dict(history=A, history_start=2 * A, prompt_len=3 * A, repetition=4 * A, presence=5 * A, frequency=6 * A, bias_token=7 * A, bias_value=8 * A, bias_start=9 * A,
            mask=10 * A, mask_row=11 * A, n_history=3, n_bias=3, n_mask_rows=1)


@pytest.mark.parametrize("change", [dict(history=None), dict(history_start=None), dict(history=None, history_start=None), dict(bias_token=None), dict(bias_value=None),
                                    dict(bias_start=None), dict(mask=None), dict(n_mask_rows=0), dict(mask_row=None), dict(n_history=-1), dict(n_bias=-1), dict(mask=A + 2), dict(repetition=A + 1)], ids=str)
def test_bad_logits_parameters(pkg, lib, change):
    p = ctypes.byref(pkg.LogitsParams(**{**GOOD, **change}))
    assert lib.htp_b200_logits_process(12 * A, 13 * A, 100, 2, 100, p, None) == -1


def test_bad_logits(pkg, lib):
    p = ctypes.byref(pkg.LogitsParams(**GOOD))
    call = lib.htp_b200_logits_process
    assert call(None, 13 * A, 100, 2, 100, p, None) == -1 and call(12 * A, None, 100, 2, 100, p, None) == -1
    assert call(12 * A, 13 * A, 100, 2, 100, None, None) == -1 and call(12 * A, 13 * A, 99, 2, 100, p, None) == -1
    assert call(12 * A, 13 * A, 100, 0, 100, p, None) == -1 and call(12 * A, 13 * A, 100, 2, 0, p, None) == -1
    assert call(12 * A + 4, 13 * A, 100, 2, 100, p, None) == -1 and call(12 * A, 12 * A + 400, 100, 2, 100, p, None) == -1


def test_no_fallback_without_a_device(pkg, lib):
    import torch
    if torch.cuda.is_available():
        pytest.skip("a GPU is present")
    assert append(pkg, lib) == -2 and attn(pkg, lib) == -2 and norm(lib) == -2
    p = ctypes.byref(pkg.LogitsParams(**GOOD))
    assert lib.htp_b200_logits_process(12 * A, 13 * A, 100, 2, 100, p, None) == -2
