"""The operators of a decoder layer in a run, as a host issues them: norm, q / k / v projections, append, attention,
output projection, norm, lm_head, logits - as requests of one message, and as direct calls captured into a graph.
Each stage is checked against its own statement in 64 bits on the buffers that the stage before it left."""
from __future__ import annotations

import ctypes

import numpy as np
import pytest
import torch

import decoder_reference as dr
from test_gpu_logits import Case, close

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def seeded():
    torch.manual_seed(1)

HIDDEN, HEADS, KV_HEADS, DIM, VOCAB, PAGE = 512, 8, 2, 64, 1024, 16


class Layer:
    def __init__(self, pkg, lib, wl, rows, lens, kv, seed):
        self.pkg, self.lib = pkg, lib
        g = torch.Generator("cuda").manual_seed(seed)
        self.cache = dr.Cache(pkg, lens, page=PAGE, heads=KV_HEADS, dim=DIM, kv=kv, seed=seed)
        self.rows = rows
        f = lambda *s: torch.randn(s, generator=g, device="cuda")  # noqa: E731
        self.t = {"x": f(rows, HIDDEN), "norm_w": 1 + 0.1 * f(HIDDEN), "norm_w2": 1 + 0.1 * f(HIDDEN), "xn": f(rows, HIDDEN) * 0, "q": f(rows, HEADS * DIM) * 0,
                  "k": f(rows, KV_HEADS * DIM) * 0, "v": f(rows, KV_HEADS * DIM) * 0, "qr": f(rows, HEADS * DIM) * 0, "att": f(rows, HEADS * DIM) * 0, "o": f(rows, HIDDEN) * 0,
                  "h": f(rows, HIDDEN) * 0, "hn": f(rows, HIDDEN) * 0, "logits": f(rows, VOCAB) * 0, "final": f(rows, VOCAB) * 0}
        a = torch.arange(64, dtype=torch.float64, device="cuda")[:, None] * 10000.0 ** (-torch.arange(0, DIM, 2, dtype=torch.float64, device="cuda") / DIM)
        self.t["rope"] = torch.cat([a.cos(), a.sin()], 1).float().contiguous()
        self.w = {}
        for i, (name, n, kk) in enumerate([("wq", HEADS * DIM, HIDDEN), ("wk", KV_HEADS * DIM, HIDDEN), ("wv", KV_HEADS * DIM, HIDDEN), ("wo", HIDDEN, HEADS * DIM), ("head", VOCAB, HIDDEN)]):
            wq, _ = wl.random_case(seed + i, 2, False, 1, kk, n)
            self.w[name] = (wq, torch.from_numpy(np.ascontiguousarray(wq)).cuda(), kk, n)
        self.case = Case(pkg, rows, VOCAB, 40, 6, [-1, 0][:1] * rows, seed)

    def matmuls(self):
        return [("wq", "xn", "q"), ("wk", "xn", "k"), ("wv", "xn", "v"), ("wo", "att", "o"), ("head", "hn", "logits")]

    def check(self, oracle, before):
        t, c = self.t, self.cache
        want = t["x"].double() / (t["x"].double().square().mean(1, keepdim=True) + 1e-5).sqrt() * t["norm_w"].double()
        assert ((t["xn"].double() - want).abs() <= 2.0 ** -19 * (want.abs() + 1e-3)).all()
        for w, src, dst in self.matmuls():
            wq, _, kk, n = self.w[w]
            ref, absdot = oracle.mul_mat_f64(t[src].cpu().numpy(), wq, n, 2, want_absdot=True)
            e = oracle.error_metrics(t[dst].cpu().numpy(), ref, absdot)
            assert e["max_rel_to_max"] <= 1e-5 and e["max_cond_rel"] <= 1e-5, (w, e)
        after = {k: (c.codes[k], c.scale[k]) for k in "kv"}  # (the buffers themselves: a graph holds their addresses)
        for k in "kv":
            c.codes[k], c.scale[k] = before[k]
        expected = dr.append(c, t["k"], t["v"], t["rope"], DIM, 2)
        for k in "kv":
            c.codes[k], c.scale[k] = after[k]
            assert torch.equal(c.scale[k], expected[k][1])
            assert torch.equal(dr.decode(c.codes[k], c.kv), dr.decode(expected[k][0], c.kv))
        pos = torch.cat([torch.arange(n - r, n, device="cuda") for r, n in c.lens])
        assert torch.equal(t["qr"].view(-1, HEADS, DIM), dr.rotate(t["q"].view(-1, HEADS, DIM), t["rope"][pos], DIM, 2))
        ref, mass, worst = dr.attention(c, t["qr"], HEADS, 0.125, 0)
        assert ((t["att"].double().view_as(ref) - ref).abs() <= dr.attention_bound(ref, mass, worst, True, c.max_ctx)).all()
        h = t["x"].double() + 0.5 * t["o"].double()
        assert ((t["h"].double() - h).abs() <= 2.0 ** -23 * (t["x"].double().abs() + t["o"].double().abs())).all()
        want = h / (h.square().mean(1, keepdim=True) + 1e-5).sqrt() * t["norm_w2"].double()
        assert ((t["hn"].double() - want).abs() <= 2.0 ** -19 * (want.abs() + 1e-2)).all()
        self.case.x = t["logits"].clone()
        want, size = self.case.want()
        close(t["final"], want, size)


def requests(layer, dev):
    """The layer's requests and the handles they name."""
    pkg, lib, c = layer.pkg, layer.lib, layer.cache
    fd = {}

    def handle(name, t):
        fd[name] = lib.htp_buf_wrap(t.data_ptr(), t.numel() * t.element_size())
        assert fd[name] > 0
        return fd[name], 0

    b = {n: handle(n, t) for n, t in layer.t.items()}
    w = {n: handle(n, v[1]) for n, v in layer.w.items()}
    kv = {"k_codes": handle("kc", c.codes["k"]), "v_codes": handle("vc", c.codes["v"]), "k_scale": handle("ks", c.scale["k"]), "v_scale": handle("vs", c.scale["v"]),
          "page_table": handle("pt", c.table), "q_start": handle("qs", c.q_start), "ctx_len": handle("cl", c.ctx_len), "n_pages": c.n_pages, "page_size": PAGE,
          "n_kv_heads": KV_HEADS, "head_dim": DIM, "kv_type": pkg.KV_I8 if c.kv == "i8" else pkg.KV_E4M3, "n_seqs": len(c.lens), "table_stride": c.table.shape[1], "n_rows": layer.rows}
    logits = {n: handle("l" + n, t) for n, t in layer.case.buf.items()}
    p = layer.case.params

    def matmul(weight, src, dst):
        _, _, kk, n = layer.w[weight]
        return pkg.pack_matmul_request(pkg.HTP_OPS_MAT_MUL_PERMUTED_W4D16A32, b[dst], b[src], w[weight], layer.rows, kk, n)

    wide = HEADS * DIM
    reqs = [pkg.pack_add_rms_norm_request(b["x"], HIDDEN, layer.rows, norm_out=b["xn"], weight=b["norm_w"]),
            matmul("wq", "xn", "q"), matmul("wk", "xn", "k"), matmul("wv", "xn", "v"),
            pkg.pack_kv_append_request(kv, b["k"], b["v"], KV_HEADS * DIM, KV_HEADS * DIM, pkg.ACT_F32, q=b["q"], q_out=b["qr"], q_stride=wide, q_out_stride=wide, n_heads=HEADS,
                                       rope_table=b["rope"], rope_mode=pkg.ROPE_HALVES, rot_dim=DIM, table_len=64),
            pkg.pack_attn_paged_request(kv, b["att"], b["qr"], wide, wide, HEADS, pkg.ACT_F32, 0.125, 0, c.max_q, c.max_ctx),
            matmul("wo", "att", "o"),
            pkg.pack_add_rms_norm_request(b["x"], HIDDEN, layer.rows, h_out=b["h"], norm_out=b["hn"], block=b["o"], weight=b["norm_w2"], block_scale=0.5),
            matmul("head", "hn", "logits"),
            pkg.pack_logits_process_request(b["final"], b["logits"], VOCAB, layer.rows, VOCAB, n_history=p.n_history, n_bias=p.n_bias, n_mask_rows=p.n_mask_rows, **logits)]
    return reqs, fd, kv, b


@pytest.mark.parametrize("kv", ["i8", "e4m3"])
@pytest.mark.parametrize("lens", [[(1, 20), (1, 1), (1, 33)], [(5, 21), (3, 3)], [(30, 30), (10, 26)]], ids=["decode", "few", "prompts"])
def test_a_layer_in_one_message(dev, oracle, wl, lens, kv):
    layer = Layer(dev.pkg, dev.lib, wl, sum(r for r, _ in lens), lens, kv, 11)
    if sum(r for r, _ in lens) > 16:
        dev.lib.htp_b200_set_option(b"a32_exact", 1)  # (the matmuls keep their 1e-5 at any token count)
    reqs, fd, _, _ = requests(layer, dev)
    before = {w: (layer.cache.codes[w].clone(), layer.cache.scale[w].clone()) for w in "kv"}
    torch.cuda.synchronize()
    chan = dev.pkg.MessageChannel(8192)
    try:
        assert chan.submit(reqs) == [0] * len(reqs)
    finally:
        chan.close()
        dev.lib.htp_b200_set_option(b"a32_exact", 0)
    layer.check(oracle, before)
    for f in fd.values():
        dev.lib.htp_buf_free(f)


def test_requests_that_are_refused(dev, wl):
    """A handle that does not exist, a region that leaves its buffer, a truncated request, arguments that the operator
    rejects: -1 for that request, the others run."""
    layer = Layer(dev.pkg, dev.lib, wl, 2, [(1, 20), (1, 5)], "i8", 12)
    pkg, lib = dev.pkg, dev.lib
    reqs, fd, kv, b = requests(layer, dev)
    small = lib.htp_buf_wrap(layer.t["x"].data_ptr(), 128)
    wide = HEADS * DIM
    good = reqs[0]
    bad = [pkg.pack_add_rms_norm_request((9999, 0), HIDDEN, 2, norm_out=b["xn"]),
           pkg.pack_add_rms_norm_request((small, 0), HIDDEN, 2, norm_out=b["xn"]),
           pkg.pack_add_rms_norm_request(b["x"], HIDDEN, 2, norm_out=(b["xn"][0], 4)),
           pkg.pack_add_rms_norm_request(None, HIDDEN, 2, norm_out=b["xn"]),
           reqs[4][:-4],
           pkg.pack_kv_append_request({**kv, "k_codes": (small, 0)}, b["k"], b["v"], 128, 128, 0),
           pkg.pack_kv_append_request({**kv, "n_pages": 2 ** 31 - 1, "n_kv_heads": 65536}, b["k"], b["v"], 128, 128, 0),
           pkg.pack_kv_append_request(kv, b["k"], b["v"], 64, 128, 0),
           pkg.pack_kv_append_request(kv, b["k"], b["v"], 128, 128, 0, rope_mode=1, rot_dim=64, table_len=2 ** 31 - 1, rope_table=b["rope"]),
           pkg.pack_attn_paged_request(kv, b["att"], b["qr"], wide, wide, 7, 0, 0.1, 0, 1, 20),
           pkg.pack_attn_paged_request(kv, b["att"], b["qr"], wide, 2 ** 31 - 4, HEADS, 0, 0.1, 0, 1, 20),
           pkg.pack_attn_paged_request(kv, b["att"], b["qr"], wide, wide, HEADS, 0, 0.1, 0, 1, 20, workspace=(small, 0), workspace_bytes=4096),
           pkg.pack_logits_process_request(b["final"], b["logits"], VOCAB, 2, VOCAB, n_mask_rows=1, mask=(small, 0), mask_row=None),
           pkg.pack_logits_process_request(b["final"], b["logits"], VOCAB - 1, 2, VOCAB)]
    torch.cuda.synchronize()
    chan = pkg.MessageChannel(8192)
    try:
        states = chan.submit([r for x in bad for r in (x, good)])
    finally:
        chan.close()
    assert states[1::2] == [0] * len(bad)
    assert states[0::2] == [-1] * len(bad)
    raw = pkg.pack_add_rms_norm_request((9999, 0), HIDDEN, 2, norm_out=b["xn"])[8:]
    buf = ctypes.create_string_buffer(raw, len(raw))
    assert lib.execute_op_simple(ctypes.cast(buf, ctypes.c_void_p)) == -1
    for f in [*fd.values(), small]:
        lib.htp_buf_free(f)


def direct(layer):
    """The same run as raw calls on torch's current stream."""
    pkg, lib, c, t = layer.pkg, layer.lib, layer.cache, layer.t
    st = dr.stream()
    p = lambda n: t[n].data_ptr()  # noqa: E731

    def matmul(weight, src, dst):
        _, w, kk, n = layer.w[weight]
        assert lib.htp_b200_mul_mat(p(dst), p(src), w.data_ptr(), layer.rows, kk, n, 2, pkg.ACT_F32, st) == 0

    wide = HEADS * DIM
    rope = pkg.Rope(table=p("rope"), positions=None, table_len=64, rot_dim=DIM, mode=pkg.ROPE_HALVES)
    assert lib.htp_b200_add_rms_norm(None, p("xn"), p("x"), None, None, None, 0, p("norm_w"), 1.0, 1e-5, HIDDEN, layer.rows, 0, st) == 0
    for w, dst in (("wq", "q"), ("wk", "k"), ("wv", "v")):
        matmul(w, "xn", dst)
    assert lib.htp_b200_kv_append(dr.ref(c.desc()), dr.ref(rope), p("k"), KV_HEADS * DIM, p("v"), KV_HEADS * DIM, p("q"), wide, p("qr"), wide, HEADS, 0, 0, st) == 0
    assert lib.htp_b200_attn_paged(p("att"), wide, p("qr"), wide, dr.ref(c.desc()), HEADS, 0, 0.125, 0, c.max_q, 64, None, 0, st) == 0
    matmul("wo", "att", "o")
    assert lib.htp_b200_add_rms_norm(p("h"), p("hn"), p("x"), p("o"), None, None, 0, p("norm_w2"), 0.5, 1e-5, HIDDEN, layer.rows, 0, st) == 0
    matmul("head", "hn", "logits")
    assert lib.htp_b200_logits_process(p("final"), p("logits"), VOCAB, layer.rows, VOCAB, dr.ref(layer.case.params), st) == 0


def test_a_captured_run_of_decoding_steps(pkg, lib, wl, oracle):
    """One graph replayed for three tokens of two sequences while the lengths grow, and two such graphs at a time on
    two streams."""
    layers = []
    for seed in (21, 22):
        lens = [(1, 30), (1, 9)]
        layer = Layer(pkg, lib, wl, 2, lens, "e4m3" if seed == 21 else "i8", seed)
        layer.cache.table = torch.tensor([[0, 1, 2, -1], [3, 4, -1, -1]], dtype=torch.int32, device="cuda")
        layer.stream = torch.cuda.Stream()
        torch.cuda.synchronize()
        with torch.cuda.stream(layer.stream):
            direct(layer)  # the matmuls make their scratch on a stream's first call
            torch.cuda.synchronize()
            layer.graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(layer.graph, stream=layer.stream):
                direct(layer)
        torch.cuda.synchronize()
        layers.append(layer)
    for step in range(1, 4):
        befores = []
        for layer in layers:
            c = layer.cache
            c.lens = [(1, 30 + step), (1, 9 + step)]
            c.max_ctx = 64
            c.ctx_len.copy_(torch.tensor([n for _, n in c.lens], dtype=torch.int32))
            layer.t["x"].normal_()
            befores.append({w: (c.codes[w].clone(), c.scale[w].clone()) for w in "kv"})
        torch.cuda.synchronize()
        for layer in layers:
            with torch.cuda.stream(layer.stream):
                layer.graph.replay()
        torch.cuda.synchronize()
        for layer, before in zip(layers, befores):
            layer.check(oracle, before)
