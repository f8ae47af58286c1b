"""Plain statements in 64 bits of the operators around a decoder's matmuls (include/htp_ops_b200.h), and
the buffers that their tests hand to the library."""
from __future__ import annotations

import ctypes
import math

import torch

CODE_MAX = {"i8": 127.0, "e4m3": 448.0}
MIN_SCALE = 2.0 ** -100


def decode(codes, kv, dtype=torch.float64):
    return codes.view(torch.int8 if kv == "i8" else torch.float8_e4m3fn).to(dtype)


def encode32(x, kv):
    """fp32 values as codes: ties to even, saturated; NaN: 0."""
    x = torch.nan_to_num(x, nan=0.0, posinf=1e6, neginf=-1e6)
    if kv == "i8":
        return torch.round(x).clamp(-127, 127).to(torch.int8).view(torch.uint8)
    return x.clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8)


class Cache:
    """A paged cache on the device with `lens` = [(rows, tokens in the cache, these rows among them)] per sequence."""

    def __init__(self, pkg, lens, *, page, heads, dim, kv, seed=1, spare=2, extra_rows=0, table_pad=1, device="cuda",
                 spread=0.5):
        self.pkg, self.lens, self.page, self.heads, self.dim, self.kv = pkg, lens, page, heads, dim, kv
        g = torch.Generator(device=device).manual_seed(seed)
        need = [-(-c // page) for _, c in lens]
        self.n_pages = sum(need) + spare
        order = torch.randperm(self.n_pages, generator=g, device=device).tolist()
        width = max(max(need), 1) + table_pad
        table, at = [], 0
        for n in need:
            table.append(order[at:at + n] + [-1] * (width - n))
            at += n
        self.table = torch.tensor(table, dtype=torch.int32, device=device)
        starts = [0]
        for q, _ in lens:
            starts.append(starts[-1] + q)
        self.starts, self.n_rows = starts, starts[-1] + extra_rows
        self.q_start = torch.tensor(starts, dtype=torch.int32, device=device)
        self.ctx_len = torch.tensor([c for _, c in lens], dtype=torch.int32, device=device)
        self.max_q = max(1, max(q for q, _ in lens))
        self.max_ctx = max(1, max(c for _, c in lens))
        shape = (self.n_pages, heads, page, dim)
        self.codes, self.scale = {}, {}
        for w in "kv":
            x = torch.randn(shape, generator=g, device=device)
            amax = x.abs().amax((2, 3))
            self.codes[w] = encode32(x * (CODE_MAX[kv] / amax)[..., None, None], kv)
            self.scale[w] = amax / CODE_MAX[kv] * torch.exp(spread * torch.randn((self.n_pages, heads), generator=g, device=device))

    def spoil_behind(self, filled):
        """No numbers (e4m3) or the largest code (signed bytes) wherever no sequence has a token."""
        used = torch.zeros((self.n_pages, self.page), dtype=torch.bool, device=self.table.device)
        for b, n in enumerate(filled):
            for p in range(-(-n // self.page)):
                used[self.table[b, p], :min(self.page, n - p * self.page)] = True
        for w in "kv":
            self.codes[w].masked_fill_(~used[:, None, :, None], 0x7F)

    def desc(self):
        p = self.pkg
        return p.PagedKv(k_codes=self.codes["k"].data_ptr(), v_codes=self.codes["v"].data_ptr(), k_scale=self.scale["k"].data_ptr(),
                         v_scale=self.scale["v"].data_ptr(), page_table=self.table.data_ptr(), q_start=self.q_start.data_ptr(),
                         ctx_len=self.ctx_len.data_ptr(), n_pages=self.n_pages, page_size=self.page, n_kv_heads=self.heads,
                         head_dim=self.dim, kv_type=p.KV_I8 if self.kv == "i8" else p.KV_E4M3, n_seqs=len(self.lens),
                         table_stride=self.table.shape[1], n_rows=self.n_rows)

    def values(self, w, b, n):
        """(heads, n, dim) in 64 bits of sequence b's first n tokens."""
        pages = self.table[b, :-(-n // self.page)].long()
        x = decode(self.codes[w][pages], self.kv) * self.scale[w][pages].double()[..., None, None]
        return x.transpose(0, 1).reshape(self.heads, -1, self.dim)[:, :n]


def attention(cache, q, n_heads, scale, window):
    """(outputs, sums of weight * |value|, largest sum of |q||k| * scale) in 64 bits, rows of the sequences."""
    group = n_heads // cache.heads
    out = torch.zeros((cache.starts[-1], n_heads, cache.dim), dtype=torch.float64, device=q.device)
    mass = torch.zeros_like(out)
    worst = torch.zeros((cache.starts[-1], n_heads, 1), dtype=torch.float64, device=q.device)
    for b, (n, c) in enumerate(cache.lens):
        if n == 0 or c == 0:
            continue
        rows = slice(cache.starts[b], cache.starts[b] + n)
        k, v = cache.values("k", b, c), cache.values("v", b, c)
        pos = torch.arange(c - n, c, device=q.device)[:, None]
        key = torch.arange(c, device=q.device)[None]
        seen = key <= pos
        if window:
            seen = seen & (key > pos - window)
        for h in range(n_heads):
            x = q[rows].double().view(n, n_heads, cache.dim)[:, h]
            s = (x @ k[h // group].T) * scale
            s = s.masked_fill(~seen, -math.inf)
            w = torch.softmax(s, 1).nan_to_num(0.0)
            out[rows, h] = w @ v[h // group]
            mass[rows, h] = w @ v[h // group].abs()
            worst[rows, h] = ((x.abs() @ k[h // group].abs().T) * scale).masked_fill(~seen, 0).amax(1, keepdim=True)
    return out, mass, worst


def attention_bound(out, mass, worst, f32, max_ctx):
    """How far the kernels' results may be off, element by element.

    A matrix instruction's fp32 accumulator is exact to one step (2^-23, truncated) per instruction.  A score is the sum of
    dim / 16 instructions for each of two fp16 terms of the query: dim / 8 steps of the sum of |q||k| it is made of (the
    terms themselves leave out 2^-22 of it).  A result is the sum of one instruction per 16 tokens and term of the
    weights, at least four warps sharing the tokens: max_ctx / 32 + 2 steps of the sum of weight * |value|.  The rest - the
    power of two (2^-22 of the instruction, 2^-20 for an argument up to 16 below the maximum), the weights' two terms
    (2^-22), joining the warps' and CTAs' sums - stays below 2^-18.  Errors of weights enter numerator and denominator:
    doubled.  fp16: the weights are rounded once (2^-11) and the result (2^-11, at least half a step of the smallest
    subnormal, 2^-25)."""
    dim = out.shape[2]
    e = mass * (2 * worst * (dim / 8 + 2) * 2.0 ** -23 + (max_ctx / 32 + 2) * 2.0 ** -23 + 2.0 ** -18)
    if not f32:
        e = e + mass * 2.0 ** -11 + out.abs() * 2.0 ** -11 + 2.0 ** -25
    return e + 1e-30


def rotate(x, table_rows, rot, mode):
    """x (rows, heads, dim) fp32; the correctly rounded fp32 steps of the library's definition."""
    if mode == 0:
        return x
    c, s = table_rows[:, None, :rot // 2], table_rows[:, None, rot // 2:]
    y = x.clone()
    a, b = (x[..., 0:rot:2], x[..., 1:rot:2]) if mode == 1 else (x[..., :rot // 2], x[..., rot // 2:rot])
    p, q = a * c - b * s, b * c + a * s
    if mode == 1:
        y[..., 0:rot:2], y[..., 1:rot:2] = p, q
    else:
        y[..., :rot // 2], y[..., rot // 2:rot] = p, q
    return y


def append(cache, k, v, rope_table, rot, mode, positions=None):
    """The cache after the step, written token by token from the definition, in fp32 steps: {"k": (codes, scale), ...}."""
    out = {w: (cache.codes[w].clone(), cache.scale[w].clone()) for w in "kv"}
    src = {"k": k.float().view(len(k), -1, cache.dim), "v": v.float().view(len(v), -1, cache.dim)}
    top = torch.tensor(CODE_MAX[cache.kv], device=k.device)
    for b, (n, c) in enumerate(cache.lens):
        for p in range((c - n) // cache.page, -(-c // cache.page)) if n else ():
            low, high = max(c - n, p * cache.page), min(c, (p + 1) * cache.page)
            page = int(cache.table[b, p])
            rows = slice(cache.starts[b] + low - (c - n), cache.starts[b] + high - (c - n))
            pos = torch.arange(low, high, device=k.device) if positions is None else positions[rows].long()
            for w in "kv":
                codes, scale = out[w]
                x = src[w][rows]
                if w == "k" and mode:
                    x = rotate(x, rope_table[pos], rot, mode)
                amax = torch.where(torch.isfinite(x), x.abs(), 0.0).amax((0, 2))
                s = torch.maximum(amax / top, torch.tensor(MIN_SCALE, device=k.device))
                if low > p * cache.page:
                    s = torch.maximum(s, scale[page])
                    old = codes[page, :, :low - p * cache.page]
                    moved = encode32(decode(old, cache.kv, torch.float32) * (scale[page] / s)[:, None, None], cache.kv)
                    codes[page, :, :low - p * cache.page] = torch.where((s > scale[page])[:, None, None], moved, old)
                scale[page] = s
                inv = torch.ones_like(s) / s
                codes[page, :, low - p * cache.page:high - p * cache.page] = encode32((x * inv[None, :, None]).transpose(0, 1), cache.kv)
    return out


def stream():
    return torch.cuda.current_stream().cuda_stream


def ref(struct):
    return ctypes.byref(struct)
