"""Cases, plain forms and calls of the operators around the quantised matmuls of a decoder:

  append     keys and values of new tokens rotated by their positions, quantised to 8 bits and put into a paged cache; the
             queries rotated in the same call
  attention  softmax attention that reads such a cache, for single tokens and for prompts
  norm       residual and norms: the block's output normed, gated, scaled and added, and the next block's input normed
  logits     penalties for repeated tokens, sparse biases and a bit mask of allowed tokens applied to logits

`own` false: elementary torch operations in 32 bits.  `own` true: the calls a program makes of the library.  Shapes are those of
the decoder stack of the benchmark (4096 wide, 32 query heads over 8 key/value heads of 128, 128256 tokens) and generic ones."""
import ctypes
import importlib
import math

import torch

own = False

MIN_SCALE = 2.0 ** -100  # what a block of zeros has as its scale
CODE_MAX = {"i8": 127.0, "e4m3": 448.0}
ACT = {"f32": torch.float32, "f16": torch.float16}


def spread(most, n, step, least=1):
    """n lengths from `least` to `most`, spread evenly in an order of their own; the first is `most`."""
    return [least + int(round((most - least) * ((1.0 - i * step) % 1.0 or 1.0))) for i in range(n)]


def lengths(case):
    """New rows and tokens in the cache (those rows among them) of every sequence."""
    b = case["seqs"]
    q = spread(case["rows"], b, 0.381966) if case["ragged"] else [case["rows"]] * b
    past = spread(case["past"], b, 0.618034, 0) if case["ragged"] else [case["past"]] * b
    return q, [i + j for i, j in zip(q, past)]


# ------------------------------------------------------------------------------------------------ the cases

def listed():
    heads = {"heads": 32, "kv_heads": 8, "dim": 128}
    cases = [
        # one user's next token, in the shapes of the benchmark's decoder
        {"name": "append 1 token", "op": "append", "seqs": 1, "rows": 1, "past": 700, "ragged": False, **heads, "page": 64, "kv": "i8", "act": "f32", "rope": "pairs", "rot": 128, "q_out": "f32"},
        # a serving step: the next token of 64 users
        {"name": "append 64 tokens", "op": "append", "seqs": 64, "rows": 1, "past": 1000, "ragged": True, **heads, "page": 64, "kv": "e4m3", "act": "f32", "rope": "halves", "rot": 128, "q_out": "f16"},
        # ragged prompts behind what the cache holds already
        {"name": "append prompts", "op": "append", "seqs": 5, "rows": 2500, "past": 333, "ragged": True, **heads, "page": 32, "kv": "e4m3", "act": "f32", "rope": "halves", "rot": 64, "q_out": "f16"},
        # one user's next token, where latency is what counts
        {"name": "attention 1 token", "op": "attention", "seqs": 1, "rows": 1, "past": 700, "ragged": False, **heads, "page": 64, "kv": "i8", "act": "f32", "window": 0},
        # a serving step: 64 users with contexts up to 8192 tokens
        {"name": "attention 64 tokens", "op": "attention", "seqs": 64, "rows": 1, "past": 8191, "ragged": True, **heads, "page": 64, "kv": "e4m3", "act": "f16", "window": 0},
        # two users deep in long documents, 8 query heads to a key/value head
        {"name": "attention long contexts", "op": "attention", "seqs": 2, "rows": 1, "past": 131071, "ragged": False, "heads": 64, "kv_heads": 8, "dim": 128, "page": 128, "kv": "i8", "act": "f32", "window": 0},
        # ragged prompts in a layer with a sliding window
        {"name": "attention prompts, window", "op": "attention", "seqs": 5, "rows": 2500, "past": 333, "ragged": True, **heads, "page": 32, "kv": "i8", "act": "f32", "window": 1024},
        # one long prompt
        {"name": "attention long prompt", "op": "attention", "seqs": 1, "rows": 8192, "past": 0, "ragged": False, **heads, "page": 64, "kv": "e4m3", "act": "f16", "window": 0},
        # between two blocks of a decoding step
        {"name": "norm 8 rows", "op": "norm", "rows": 8, "n": 4096, "post": True, "gate": "shared", "norm": "f16"},
        # the same over a prompt; an odd number of rows
        {"name": "norm prompt", "op": "norm", "rows": 8191, "n": 4096, "post": True, "gate": "rows", "norm": "f32"},
        # a single user's logits
        {"name": "logits 1 row", "op": "logits", "rows": 1, "vocab": 128256, "history": 4096, "biases": 50, "mask": False},
        # a serving step's logits, some rows bound to a grammar
        {"name": "logits 200 rows", "op": "logits", "rows": 200, "vocab": 128256, "history": 2000, "biases": 300, "mask": True},
    ]
    return cases


def log_uniform(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(("append", "attention", "attention", "norm", "logits"))
    if op == "norm":
        n = log_uniform(rng, 64, 16384)
        return {"op": op, "rows": log_uniform(rng, 1, max(2, 33000000 // n)), "n": n, "post": rng.random() < 0.5,
                "gate": rng.choice(("none", "shared", "rows")), "norm": rng.choice(("f32", "f16"))}
    if op == "logits":
        vocab = log_uniform(rng, 500, 200000)
        return {"op": op, "rows": log_uniform(rng, 1, max(2, min(1000, 25000000 // vocab))), "vocab": vocab, "history": log_uniform(rng, 1, 8000),
                "biases": log_uniform(rng, 1, min(300, vocab // 2)), "mask": rng.random() < 0.5}
    kv_heads = rng.choice((1, 2, 4, 8))
    case = {"op": op, "heads": kv_heads * rng.choice((1, 2, 3, 4, 7, 8)), "kv_heads": kv_heads, "dim": rng.choice((64, 128)), "page": rng.choice((16, 32, 64, 128)),
            "kv": rng.choice(("i8", "e4m3")), "act": rng.choice(("f32", "f16")), "ragged": rng.random() < 0.7}
    wide = case["heads"] * case["dim"]
    if rng.random() < 0.5:  # decoding, up to four rows a sequence
        case["seqs"], case["rows"] = log_uniform(rng, 1, 100), rng.choice((1, 1, 1, 2, 4))
        case["past"] = log_uniform(rng, 1, min(60000, 200000000 // (case["seqs"] * kv_heads * case["dim"])))
    else:
        case["seqs"] = log_uniform(rng, 1, 8)
        case["rows"] = log_uniform(rng, 2, min(6000, 30000000 // wide // case["seqs"]))
        case["past"] = log_uniform(rng, 1, 2000)
    if op == "append":
        case.update(rope=rng.choice(("none", "pairs", "halves")), rot=rng.choice((32, 64)), q_out=rng.choice(("f32", "f16")))
    else:
        case["window"] = 0 if rng.random() < 0.7 else log_uniform(rng, 8, 4000)
        case["rows"] = min(case["rows"], int(1.5e9 / (case["seqs"] * case["heads"] * (case["rows"] + case["past"]))) or 1)
    return case


# ------------------------------------------------------------------------------------------------ their inputs

def to_codes(x, kv):
    if kv == "i8":
        return torch.round(x).clamp(-127, 127).to(torch.int8).view(torch.uint8)
    return x.clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8)


def from_codes(codes, kv, dtype):
    return codes.view(torch.int8 if kv == "i8" else torch.float8_e4m3fn).to(dtype)


def a_cache(case, gen, q_lens, ctx_lens, filled):
    """Pages in an order of their own, `filled[i]` tokens of sequence i in them; what lies behind is whatever was there."""
    page, heads, dim, kv = case["page"], case["kv_heads"], case["dim"], case["kv"]
    need = [-(-c // page) for c in ctx_lens]
    n_pages = sum(need) + 3
    order = torch.randperm(n_pages, generator=gen, device="cuda").to(torch.int32)
    width = max(need) + 1
    at = torch.tensor([sum(need[:i]) for i in range(len(need))], device="cuda").unsqueeze(1) + torch.arange(width, device="cuda")
    held = torch.arange(width, device="cuda") < torch.tensor(need, device="cuda").unsqueeze(1)
    table = torch.where(held, order[at.clamp(max=n_pages - 1)], -1).contiguous()
    s = {"page_table": table, "n_pages": n_pages,
         "q_start": torch.tensor([sum(q_lens[:i]) for i in range(len(q_lens) + 1)], dtype=torch.int32, device="cuda"),
         "ctx_len": torch.tensor(ctx_lens, dtype=torch.int32, device="cuda"), "n_rows": sum(q_lens), "max_q": max(q_lens), "max_ctx": max(ctx_lens)}
    in_use = torch.zeros((n_pages, page), dtype=torch.bool, device="cuda")
    tok = torch.arange(width * page, device="cuda").view(width, page)
    use = tok.unsqueeze(0) < torch.tensor(filled, device="cuda").view(-1, 1, 1)
    in_use[table[held].long()] = use[held]
    for which in ("k", "v"):
        codes = torch.empty((n_pages, heads, page, dim), dtype=torch.uint8, device="cuda")
        scale = torch.empty((n_pages, heads), dtype=torch.float32, device="cuda")
        for p in range(0, n_pages, 4096):
            x = torch.randn((min(4096, n_pages - p), heads, page, dim), generator=gen, device="cuda")
            size = torch.exp(0.5 * torch.randn((len(x), heads), generator=gen, device="cuda"))
            amax = x.abs().amax((2, 3))
            codes[p:p + len(x)] = to_codes(x * (CODE_MAX[kv] / amax)[:, :, None, None], kv)
            scale[p:p + len(x)] = amax * size / CODE_MAX[kv]
        codes.masked_fill_(~in_use[:, None, :, None], 0x7F)  # (no number, in e4m3)
        s[which + "_codes"], s[which + "_scale"] = codes, scale
    return s


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    s = {"case": case}

    def normal(*shape, dtype=torch.float32):
        return torch.randn(shape, generator=gen, device="cuda").to(dtype)

    if case["op"] == "norm":
        rows, n = case["rows"], case["n"]
        s.update(x=normal(rows, n) * 3, block=normal(rows, n), weight=1 + 0.1 * normal(n), post=1 + 0.1 * normal(n) if case["post"] else None, block_scale=0.7, eps=1e-5,
                 gate={"none": None, "shared": normal(1, n), "rows": None}[case["gate"]], h=torch.empty((rows, n), device="cuda"),
                 out=torch.empty((rows, n), dtype=ACT[case["norm"]], device="cuda"))
        if case["gate"] == "rows":
            s["gate"] = normal(rows, n)
        return s
    if case["op"] == "logits":
        rows, vocab = case["rows"], case["vocab"]
        hist = spread(case["history"], rows, 0.618034, 0)
        biases = spread(case["biases"], rows, 0.381966, 0)
        ints = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
        starts = lambda v: ints([0] + torch.tensor(v).cumsum(0).tolist())  # noqa: E731
        # texts repeat themselves: tokens drawn from a skewed distribution
        tokens = (vocab * torch.rand(sum(hist), generator=gen, device="cuda") ** 4).to(torch.int32).clamp(max=vocab - 1)
        first = torch.randint(0, vocab, (rows, 1), generator=gen, device="cuda")
        take = torch.arange(case["biases"], device="cuda") < ints(biases).unsqueeze(1)
        s.update(logits=4 * normal(rows, vocab), out=torch.empty((rows, vocab), device="cuda"), history=tokens, history_start=starts(hist), prompt_len=ints([h // 2 for h in hist]),
                 repetition=1 + 0.5 * torch.rand(rows, generator=gen, device="cuda"), presence=torch.rand(rows, generator=gen, device="cuda"),
                 frequency=0.3 * torch.rand(rows, generator=gen, device="cuda"), bias_start=starts(biases),
                 bias_token=((first + torch.arange(case["biases"], device="cuda") * (vocab // max(1, case["biases"]))) % vocab)[take].to(torch.int32),
                 bias_value=3 * normal(rows, case["biases"])[take], mask=None, mask_row=None)
        if case["mask"]:  # two grammars; every third row is free
            words = -(-vocab // 32)
            bits = torch.randint(-2 ** 31, 2 ** 31, (2, words), generator=gen, device="cuda").to(torch.int32)
            bits[1] &= torch.randint(-2 ** 31, 2 ** 31, (4, words), generator=gen, device="cuda").to(torch.int32).amin(0)
            s.update(mask=bits.contiguous(), mask_row=ints([i % 3 - 1 for i in range(rows)]))
        return s
    q_lens, ctx_lens = lengths(case)
    dim, act = case["dim"], ACT[case["act"]]
    rows = sum(q_lens)
    append = case["op"] == "append"
    s.update(a_cache(case, gen, q_lens, ctx_lens, [c - q for c, q in zip(ctx_lens, q_lens)] if append else ctx_lens))
    if append:
        # the three lie side by side, as the output of one matrix does
        wide = normal(rows, (case["heads"] + 2 * case["kv_heads"]) * dim, dtype=act)
        s["q"], s["k"], s["v"] = wide.split([case["heads"] * dim, case["kv_heads"] * dim, case["kv_heads"] * dim], dim=1)
        s["q_out"] = torch.empty((rows, case["heads"] * dim), dtype=ACT[case["q_out"]], device="cuda")
        angle = torch.arange(max(ctx_lens), device="cuda", dtype=torch.float64).unsqueeze(1) * 500000.0 ** (-torch.arange(0, case["rot"], 2, device="cuda", dtype=torch.float64) / case["rot"])
        s["rope_table"] = torch.cat([angle.cos(), angle.sin()], 1).float().contiguous()
    else:
        s["q"] = normal(rows, case["heads"] * dim, dtype=act) * 1.5
        s["out"] = torch.empty_like(s["q"])
        s["scale"] = dim ** -0.5
        s["workspace"] = torch.zeros(64 << 20, dtype=torch.uint8, device="cuda")  # a program has one for all its calls
    return s


# ------------------------------------------------------------------------------------------------ the plain forms

def of_rows(s):
    """Sequence and position in the cache of every row."""
    row = torch.arange(s["n_rows"], device="cuda", dtype=torch.int32)
    seq = torch.searchsorted(s["q_start"], row, right=True) - 1
    q_len = s["q_start"][1:] - s["q_start"][:-1]
    return seq, (s["ctx_len"] - q_len)[seq] + row - s["q_start"][seq]


def rotated(x, table, rope, rot):
    """x: (rows, heads, dim) in 32 bits; table: (rows, rot), cosines and then sines."""
    if rope == "none":
        return x
    c, n = table[:, None, :rot // 2], table[:, None, rot // 2:]
    r = x[..., :rot]
    a, b = (r[..., 0::2], r[..., 1::2]) if rope == "pairs" else (r[..., :rot // 2], r[..., rot // 2:])
    y, z = a * c - b * n, b * c + a * n
    r = torch.stack([y, z], -1).flatten(-2) if rope == "pairs" else torch.cat([y, z], -1)
    return torch.cat([r, x[..., rot:]], -1)


def plain_append(s):
    case = s["case"]
    page, heads, dim, kv = case["page"], case["kv_heads"], case["dim"], case["kv"]
    seq, pos = of_rows(s)
    table = s["rope_table"][pos.long()]
    pages, slot = s["page_table"][seq, (pos // page).long()].long(), (pos % page).long()
    q = rotated(s["q"].float().view(-1, case["heads"], dim), table, case["rope"], case["rot"])
    first = s["ctx_len"] - (s["q_start"][1:] - s["q_start"][:-1])  # the first new token of each sequence
    at = torch.arange(len(first), device="cuda")
    old_page, old = s["page_table"][at, (first // page).long()].long(), torch.arange(page, device="cuda") < (first % page).unsqueeze(1)
    for which in ("k", "v"):
        x = s[which].float().view(-1, heads, dim)
        if which == "k":
            x = rotated(x, table, case["rope"], case["rot"])
        codes, scale = s[which + "_codes"], s[which + "_scale"]
        amax = torch.zeros_like(scale).scatter_reduce(0, pages.unsqueeze(1).expand(-1, heads), x.abs().amax(2), "amax")
        fresh = (amax / torch.full_like(amax, CODE_MAX[kv])).clamp(min=MIN_SCALE)
        before = scale[old_page]  # of the pages that hold older tokens already
        after = torch.where(old[:, :1], torch.maximum(before, fresh[old_page]), fresh[old_page])
        values = from_codes(codes[old_page], kv, torch.float32) * torch.where(old[:, :1], before / after, 1.0)[:, :, None, None]
        codes[old_page] = torch.where(old[:, None, :, None], to_codes(values, kv), codes[old_page])
        scale[pages] = fresh[pages]
        scale[old_page] = after
        codes[pages, :, slot] = to_codes(x * (1.0 / scale[pages]).unsqueeze(2), kv)
    return q.flatten(1).to(ACT[case["q_out"]])


def plain_attention(s):
    case = s["case"]
    page, heads, dim, kv, group = case["page"], case["kv_heads"], case["dim"], case["kv"], case["heads"] // case["kv_heads"]
    n, most = len(s["ctx_len"]), s["max_ctx"]
    wide = -(-most // page)
    pages = s["page_table"][:, :wide].long().clamp(min=0)
    key = torch.arange(wide * page, device="cuda")
    held = key < s["ctx_len"].unsqueeze(1)

    def values(which):
        x = from_codes(s[which + "_codes"][pages], kv, torch.float32) * s[which + "_scale"][pages][..., None, None]  # (n, wide, heads, page, dim)
        x = x.permute(0, 2, 1, 3, 4).reshape(n, heads, wide * page, dim)
        return torch.where(held[:, None, :, None], x, 0.0)

    seq, pos = of_rows(s)
    row = torch.arange(s["n_rows"], device="cuda") - s["q_start"][seq]
    q = torch.zeros((n, s["max_q"], case["heads"] * dim), device="cuda")
    q[seq, row] = s["q"].float()
    q = q.view(n, s["max_q"], heads, group, dim).permute(0, 2, 3, 1, 4).reshape(n, heads, group * s["max_q"], dim)
    at = torch.zeros((n, s["max_q"]), dtype=torch.int64, device="cuda")
    at[seq, row] = pos.long()
    seen = (key <= at.unsqueeze(2)) & held.unsqueeze(1)
    if case["window"]:
        seen &= key > at.unsqueeze(2) - case["window"]
    score = (torch.matmul(q, values("k").transpose(2, 3)) * s["scale"]).view(n, heads, group, s["max_q"], -1)
    score.masked_fill_(~seen[:, None, None], -math.inf)
    score -= score.amax(-1, keepdim=True).clamp(min=-3e38)
    score.exp_()
    total = score.sum(-1)
    out = torch.matmul(score.view(n, heads, group * s["max_q"], -1), values("v")).view(n, heads, group, s["max_q"], dim) / total.unsqueeze(-1)
    return out.permute(0, 3, 1, 2, 4).reshape(n, s["max_q"], -1)[seq, row].to(s["q"].dtype)


def plain_norm(s):
    b = s["block"]
    if s["post"] is not None:
        b = b * torch.rsqrt(b.square().mean(1, keepdim=True) + s["eps"]) * s["post"]
    if s["gate"] is not None:
        b = b * s["gate"]
    h = s["x"] + s["block_scale"] * b
    return h, (h * torch.rsqrt(h.square().mean(1, keepdim=True) + s["eps"]) * s["weight"]).to(s["out"].dtype)


def plain_logits(s):
    x, (rows, vocab) = s["logits"], s["logits"].shape
    at = torch.arange(len(s["history"]), device="cuda", dtype=torch.int32)
    row = torch.searchsorted(s["history_start"], at, right=True) - 1
    answer = at - s["history_start"][row] >= s["prompt_len"][row]
    place = row * vocab + s["history"]
    count = torch.zeros(rows * vocab, device="cuda").index_add_(0, place, answer.float()).view(rows, vocab)
    seen = torch.zeros(rows * vocab, dtype=torch.bool, device="cuda").index_fill_(0, place, True).view(rows, vocab)
    rep = s["repetition"].unsqueeze(1)
    y = torch.where(seen, torch.where(x > 0, x / rep, x * rep), x)
    y = y - s["frequency"].unsqueeze(1) * count - s["presence"].unsqueeze(1) * (count > 0)
    row = torch.searchsorted(s["bias_start"], torch.arange(len(s["bias_token"]), device="cuda", dtype=torch.int32), right=True) - 1
    y = y.view(-1).index_add(0, row * vocab + s["bias_token"], s["bias_value"]).view(rows, vocab)
    if s["mask"] is not None:
        token = torch.arange(vocab, device="cuda")
        allowed = (s["mask"][:, token // 32] >> (token % 32)) & 1
        y = torch.where((allowed[s["mask_row"].clamp(min=0).long()] == 1) | (s["mask_row"] < 0).unsqueeze(1), y, -math.inf)
    return y


# ------------------------------------------------------------------------------------------------ the library's calls

def library():
    pkg = importlib.import_module("htp-ops-lib_b200")
    return pkg, pkg.load()


def ptr(t):
    return None if t is None else t.data_ptr()


def handles(s):
    """What a program makes once for its cache and its steps: descriptors of the buffers that it holds."""
    pkg, lib = library()
    case = s["case"]
    made = {"lib": lib, "pkg": pkg}
    if case["op"] in ("append", "attention"):
        made["kv"] = pkg.PagedKv(k_codes=ptr(s["k_codes"]), v_codes=ptr(s["v_codes"]), k_scale=ptr(s["k_scale"]), v_scale=ptr(s["v_scale"]), page_table=ptr(s["page_table"]),
                                 q_start=ptr(s["q_start"]), ctx_len=ptr(s["ctx_len"]), n_pages=s["n_pages"], page_size=case["page"], n_kv_heads=case["kv_heads"],
                                 head_dim=case["dim"], kv_type=pkg.KV_I8 if case["kv"] == "i8" else pkg.KV_E4M3, n_seqs=len(s["ctx_len"]),
                                 table_stride=s["page_table"].shape[1], n_rows=s["n_rows"])
        made["kv_ref"] = ctypes.byref(made["kv"])
    if case["op"] == "append":
        mode = {"none": pkg.ROPE_NONE, "pairs": pkg.ROPE_PAIRS, "halves": pkg.ROPE_HALVES}[case["rope"]]
        made["rope"] = pkg.Rope(table=ptr(s["rope_table"]), positions=None, table_len=len(s["rope_table"]), rot_dim=case["rot"], mode=mode)
        made["rope_ref"] = ctypes.byref(made["rope"])
    if case["op"] == "logits":
        made["params"] = pkg.LogitsParams(history=ptr(s["history"]), history_start=ptr(s["history_start"]), prompt_len=ptr(s["prompt_len"]), repetition=ptr(s["repetition"]),
                                          presence=ptr(s["presence"]), frequency=ptr(s["frequency"]), bias_token=ptr(s["bias_token"]), bias_value=ptr(s["bias_value"]),
                                          bias_start=ptr(s["bias_start"]), mask=ptr(s["mask"]), mask_row=ptr(s["mask_row"]), n_history=len(s["history"]),
                                          n_bias=len(s["bias_token"]), n_mask_rows=0 if s["mask"] is None else len(s["mask"]))
        made["params_ref"] = ctypes.byref(made["params"])
    return made


def call(s):
    if "handles" not in s:
        s["handles"] = handles(s)
    made, case = s["handles"], s["case"]
    pkg, lib = made["pkg"], made["lib"]
    stream = torch.cuda.current_stream().cuda_stream
    if case["op"] == "append":
        act = pkg.ACT_F32 if case["act"] == "f32" else pkg.ACT_F16
        rc = lib.htp_b200_kv_append(made["kv_ref"], made["rope_ref"], s["k"].data_ptr(), s["k"].stride(0), s["v"].data_ptr(), s["v"].stride(0), s["q"].data_ptr(), s["q"].stride(0),
                                    s["q_out"].data_ptr(), s["q_out"].stride(0), case["heads"], act, pkg.ACT_F32 if case["q_out"] == "f32" else pkg.ACT_F16, stream)
    elif case["op"] == "attention":
        rc = lib.htp_b200_attn_paged(s["out"].data_ptr(), s["out"].stride(0), s["q"].data_ptr(), s["q"].stride(0), made["kv_ref"], case["heads"],
                                     pkg.ACT_F32 if case["act"] == "f32" else pkg.ACT_F16, s["scale"], case["window"], s["max_q"], s["max_ctx"], s["workspace"].data_ptr(),
                                     s["workspace"].numel(), stream)
    elif case["op"] == "norm":
        rc = lib.htp_b200_add_rms_norm(s["h"].data_ptr(), s["out"].data_ptr(), s["x"].data_ptr(), s["block"].data_ptr(), ptr(s["post"]), ptr(s["gate"]),
                                       case["n"] if case["gate"] == "rows" else 0, s["weight"].data_ptr(), s["block_scale"], s["eps"], case["n"], case["rows"],
                                       pkg.ACT_F32 if case["norm"] == "f32" else pkg.ACT_F16, stream)
    else:
        rc = lib.htp_b200_logits_process(s["out"].data_ptr(), s["logits"].data_ptr(), case["vocab"], case["rows"], case["vocab"], made["params_ref"], stream)
    if rc != 0:
        raise RuntimeError("%s: the library answers %d" % (case["op"], rc))


def run(s):
    op = s["case"]["op"]
    if own:
        call(s)
        got = {"append": ("q_out",), "attention": ("out",), "norm": ("h", "out"), "logits": ("out",)}[op]
        got = [s[name] for name in got]
    else:
        got = {"append": plain_append, "attention": plain_attention, "norm": plain_norm, "logits": plain_logits}[op](s)
        got = list(got) if isinstance(got, tuple) else [got]
    if op == "append":  # the cache after it: 8-bit numbers and their scales
        kind = torch.int8 if s["case"]["kv"] == "i8" else torch.float8_e4m3fn
        got += [s["k_codes"].view(kind), s["v_codes"].view(kind), s["k_scale"], s["v_scale"]]
    return got


# ------------------------------------------------------------------------------------------------ their floors

def work(case):
    if case["op"] == "norm":
        n = case["rows"] * case["n"]
        gate = {"none": 0, "shared": 4 * case["n"], "rows": 4 * n}[case["gate"]]
        return {"bytes": 12 * n + (4 if case["norm"] == "f32" else 2) * n + gate + (8 if case["post"] else 4) * case["n"], "flops": 12 * n}
    if case["op"] == "logits":
        rows, vocab = case["rows"], case["vocab"]
        hist, biases = sum(spread(case["history"], rows, 0.618034, 0)), sum(spread(case["biases"], rows, 0.381966, 0))
        return {"bytes": 8 * rows * vocab + 4 * hist + 8 * biases + 28 * rows + (vocab // 4 if case["mask"] else 0), "flops": 4 * (hist + biases)}
    q_lens, ctx_lens = lengths(case)
    heads, dim, size = case["kv_heads"], case["dim"], 4 if case["act"] == "f32" else 2
    rows = sum(q_lens)
    if case["op"] == "append":
        wide = rows * (case["heads"] + 2 * heads) * dim
        pages = sum(-(-c // case["page"]) - (c - q) // case["page"] for q, c in zip(q_lens, ctx_lens))
        out = rows * case["heads"] * dim * (4 if case["q_out"] == "f32" else 2) + 2 * rows * heads * dim + 16 * pages * heads
        return {"bytes": wide * size + out + (0 if case["rope"] == "none" else 4 * rows * case["rot"]) + 4 * pages, "flops": 6 * wide}
    window = case["window"] or 1 << 40
    pairs = keys = 0
    for q, c in zip(q_lens, ctx_lens):
        full = max(0, min(q, c - window + 1))  # rows that see a whole window
        pairs += full * min(window, c) + sum(range(c - q + 1, c - full + 1)) if window <= c else sum(range(c - q + 1, c + 1))
        keys += min(c, window + q - 1)
    return {"bytes": 2 * rows * case["heads"] * dim * size + keys * heads * 2 * (dim + 4 / case["page"]) + 4 * keys / case["page"], "flops": 4 * dim * case["heads"] * pairs}


# ------------------------------------------------------------------------------------------------ from the definitions, in 64 bits

def exact_rotation(x, angles, rope, rot):
    """(rows, heads, dim) as complex numbers turned by their angles; `angles` complex, (rows, rot / 2)."""
    if rope == "none":
        return x
    head = x[..., :rot]
    z = torch.view_as_complex(head.reshape(*head.shape[:-1], rot // 2, 2)) if rope == "pairs" else torch.complex(head[..., :rot // 2].contiguous(), head[..., rot // 2:].contiguous())
    z = z * angles.unsqueeze(1)
    y = x.clone()
    if rope == "pairs":
        y[..., 0:rot:2], y[..., 1:rot:2] = z.real, z.imag
    else:
        y[..., :rot // 2], y[..., rot // 2:rot] = z.real, z.imag
    return y


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "norm":
        b, x = s["block"].double(), s["x"].double()
        rms = lambda t: (t.pow(2).sum(1, keepdim=True) / t.shape[1] + s["eps"]).sqrt()  # noqa: E731
        if s["post"] is not None:
            b = b / rms(b) * s["post"].double()
        h = x + s["block_scale"] * b * (1.0 if s["gate"] is None else s["gate"].double())
        return [h, h / rms(h) * s["weight"].double()]
    if case["op"] == "logits":
        y = s["logits"].double()
        hist, start, split = s["history"].long(), s["history_start"].tolist(), s["prompt_len"].tolist()
        bias_start = s["bias_start"].tolist()
        for r in range(case["rows"]):
            rep, fre, pre = (float(s[name][r]) for name in ("repetition", "frequency", "presence"))
            mine = hist[start[r]:start[r + 1]]
            every = torch.bincount(mine, minlength=case["vocab"])
            answer = torch.bincount(mine[split[r]:], minlength=case["vocab"])
            y[r] *= torch.where(every > 0, torch.where(y[r] > 0, 1.0 / rep, rep), 1.0)
            y[r] -= fre * answer + pre * (answer > 0)
            here = slice(bias_start[r], bias_start[r + 1])
            y[r, s["bias_token"][here].long()] += s["bias_value"][here].double()
            if s["mask"] is not None and int(s["mask_row"][r]) >= 0:
                bits = (s["mask"][int(s["mask_row"][r])].unsqueeze(1) >> torch.arange(32, device="cuda")) & 1
                y[r, bits.flatten()[:case["vocab"]] == 0] = -math.inf
        return [y]
    q_lens, ctx_lens = lengths(case)
    heads, dim, page, kv = case["kv_heads"], case["dim"], case["page"], case["kv"]
    if case["op"] == "append":
        half = case["rot"] // 2
        angles = torch.complex(s["rope_table"][:, :half].double(), s["rope_table"][:, half:].double())
        q = s["q"].double().view(-1, case["heads"], dim)
        new = {"k": s["k"].double().view(-1, heads, dim), "v": s["v"].double().view(-1, heads, dim)}
        outs, begin = {"q": []}, 0
        state = {w: (from_codes(s[w + "_codes"], kv, torch.float64), s[w + "_scale"].double()) for w in ("k", "v")}
        for i, (n, c) in enumerate(zip(q_lens, ctx_lens)):
            rows, turn = slice(begin, begin + n), angles[c - n:c]
            outs["q"].append(exact_rotation(q[rows], turn, case["rope"], case["rot"]))
            new["k"][rows] = exact_rotation(new["k"][rows], turn, case["rope"], case["rot"])
            for p in range((c - n) // page, (c - 1) // page + 1):
                low, high = max(c - n, p * page), min(c, (p + 1) * page)
                at = int(s["page_table"][i, p])
                for w in ("k", "v"):
                    codes, scale = state[w]
                    x = new[w][begin + low - (c - n):begin + high - (c - n)].transpose(0, 1)
                    wanted = (x.abs().amax((1, 2)) / CODE_MAX[kv]).clamp(min=MIN_SCALE)
                    if low > p * page:
                        wanted = torch.maximum(wanted, scale[at])
                        held = codes[at, :, :low - p * page] * (scale[at] / wanted)[:, None, None]
                        codes[at, :, :low - p * page] = from_codes(to_codes(held, kv), kv, torch.float64)
                    codes[at, :, low - p * page:high - p * page] = from_codes(to_codes(x / wanted[:, None, None], kv), kv, torch.float64)
                    scale[at] = wanted
            begin += n
        codes = [state[w][0] if kv == "e4m3" else None for w in ("k", "v")]  # (whole numbers are compared as such)
        return [torch.cat(outs["q"]).flatten(1), *codes, state["k"][1], state["v"][1]]
    out, begin, group = [], 0, case["heads"] // heads
    for i, (n, c) in enumerate(zip(q_lens, ctx_lens)):
        pages = s["page_table"][i, :-(-c // page)].long()
        k, v = ((from_codes(s[w + "_codes"][pages], kv, torch.float64) * s[w + "_scale"][pages].double()[:, :, None, None]).transpose(0, 1).reshape(heads, -1, dim)[:, :c] for w in ("k", "v"))
        query = s["q"][begin:begin + n].double().view(n, heads, group, dim)
        ahead = torch.arange(c, device="cuda") - torch.arange(c - n, c, device="cuda").unsqueeze(1)
        hidden = (ahead > 0) | (ahead <= -case["window"] if case["window"] else False)
        got = torch.empty_like(query)
        for h in range(heads):
            for g in range(group):
                score = (query[:, h, g] @ k[h].T * s["scale"]).masked_fill_(hidden, -math.inf)
                got[:, h, g] = torch.softmax(score, 1) @ v[h]
        out.append(got.flatten(1))
        begin += n
    return [torch.cat(out)]
