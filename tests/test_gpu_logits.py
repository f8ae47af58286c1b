"""Logits processing against a statement in 64 bits, token by token."""
from __future__ import annotations

import math

import pytest
import torch

import decoder_reference as dr

pytestmark = pytest.mark.gpu


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


class Case:
    def __init__(self, pkg, rows, vocab, hist, biases, mask_row, seed, stride=None):
        g = torch.Generator().manual_seed(seed)
        rnd = lambda n: torch.randint(0, n, (1,), generator=g).item()  # noqa: E731
        self.rows, self.vocab, self.stride = rows, vocab, stride or vocab
        self.hist = [[rnd(vocab) if rnd(3) else rnd(min(vocab, 5)) for _ in range(hist if r % 3 else hist // 2)] for r in range(rows)]
        if self.hist[0]:
            self.hist[0][:3] = [-1, vocab, 2 ** 31 - 1][:len(self.hist[0])]  # count for nothing
        self.prompt = [len(h) // (1 + r % 3) if r % 4 else 0 for r, h in enumerate(self.hist)]
        self.bias = [[(rnd(vocab) if rnd(4) else 1 % vocab, rnd(2000) / 300.0 - 3) for _ in range(biases if r % 2 else biases // 3)] for r in range(rows)]
        if self.bias[-1]:
            self.bias[-1][0] = (-5, 100.0)
        self.rep, self.pres, self.freq = (torch.rand(rows, generator=g).cuda() * s + o for s, o in ((1.0, 0.6), (1.0, -0.3), (0.5, 0.0)))
        self.mask_row = mask_row
        n_masks = max([m for m in mask_row or [0]] + [0]) + 1
        self.bits = torch.rand((n_masks, vocab), generator=g).cuda() < 0.4
        if n_masks > 1:
            self.bits[1] = False  # nothing is allowed
        words = -(-vocab // 32)
        padded = torch.zeros((n_masks, words * 32), dtype=torch.int64, device="cuda")
        padded[:, :vocab] = self.bits
        packed = (padded.view(n_masks, words, 32) << torch.arange(32, device="cuda")).sum(2)
        packed = torch.where(packed >= 2 ** 31, packed - 2 ** 32, packed).to(torch.int32)
        starts = lambda v: ints([0] + torch.tensor([len(x) for x in v]).cumsum(0).tolist())  # noqa: E731
        self.buf = {"history": ints(sum(self.hist, []) or [0]), "history_start": starts(self.hist), "prompt_len": ints(self.prompt),
                    "repetition": self.rep, "presence": self.pres, "frequency": self.freq, "bias_token": ints([t for b in self.bias for t, _ in b] or [0]),
                    "bias_value": torch.tensor([v for b in self.bias for _, v in b] or [0.0], dtype=torch.float32, device="cuda"), "bias_start": starts(self.bias)}
        if mask_row is not None:
            self.buf["mask"], self.buf["mask_row"] = packed.contiguous(), ints(mask_row)
        self.params = pkg.LogitsParams(n_history=sum(map(len, self.hist)), n_bias=sum(map(len, self.bias)), n_mask_rows=n_masks,
                                       **{k: v.data_ptr() for k, v in self.buf.items()})
        self.x = torch.randn((rows, self.stride), generator=g).cuda() * 4
        self.x[0, 0] = 0.0
        if vocab > 4:
            self.x[rows - 1, 3], self.x[0, 2] = -math.inf, math.inf

    def want(self):
        y = self.x[:, :self.vocab].double().cpu()
        values = self.buf["bias_value"].double().cpu().tolist()
        at = 0
        rep, pres, freq = (t.double().cpu().tolist() for t in (self.rep, self.pres, self.freq))
        size = y.abs()
        for r in range(self.rows):
            count, seen = {}, set()
            for i, t in enumerate(self.hist[r]):
                if 0 <= t < self.vocab:
                    seen.add(t)
                    if i >= self.prompt[r]:
                        count[t] = count.get(t, 0) + 1
            for t in seen:
                v = y[r, t].item()
                v = v / rep[r] if v > 0 else v * rep[r]
                size[r, t] += abs(v)
                y[r, t] = v - freq[r] * count.get(t, 0) - pres[r] * (t in count)
                size[r, t] += abs(freq[r]) * count.get(t, 0) + abs(pres[r])
            for t, _ in self.bias[r]:
                if 0 <= t < self.vocab:
                    y[r, t] += values[at]
                    size[r, t] += abs(values[at]) * max(8, len(self.bias[r]) / 8)  # (a sum of up to so many)
                at += 1
            if self.mask_row is not None and self.mask_row[r] >= 0:
                y[r, ~self.bits[self.mask_row[r]].cpu()] = -math.inf
        return y.cuda(), size.cuda()

    def run(self, lib, dst, src):
        return lib.htp_b200_logits_process(dst.data_ptr(), src.data_ptr(), self.stride, self.rows, self.vocab, dr.ref(self.params), dr.stream())


def close(got, want, size):
    fine = torch.isfinite(want)
    assert torch.equal(got[~fine].double(), want[~fine])
    # at most 6 + (biases of a token) roundings of terms that `size` adds up
    err = (got.double() - want).abs()[fine]
    assert (err <= 2.0 ** -24 * 8 * size[fine]).all(), (err / size[fine]).max()


@pytest.mark.parametrize("rows,vocab,hist,biases,stride", [(1, 1, 3, 2, None), (1, 128256, 4096, 50, None), (3, 1000, 700, 33, None), (7, 4099, 50, 300, None),
                                                           (9, 5003, 0, 0, None), (6, 8191, 1500, 5, 8200), (160, 32001, 60, 40, None), (2, 31, 64, 3, 33), (3, 700, 10, 900, None)])
@pytest.mark.parametrize("masked", [False, True])
def test_matches_64_bits(pkg, lib, rows, vocab, hist, biases, stride, masked):
    mask_row = [[-1, 0, 1, 2][r % 4] for r in range(rows)] if masked else None
    c = Case(pkg, rows, vocab, hist, biases, mask_row, seed=vocab + rows, stride=stride)
    want, size = c.want()
    out = torch.full_like(c.x, 7.0)
    assert c.run(lib, out, c.x) == 0
    close(out[:, :vocab], want, size)
    assert (out[:, vocab:] == 7.0).all()
    behind = c.x[:, vocab:].clone()
    assert c.run(lib, c.x, c.x) == 0  # in place
    assert torch.equal(c.x[:, :vocab].nan_to_num(1e9), out[:, :vocab].nan_to_num(1e9)) and torch.equal(c.x[:, vocab:], behind)
    assert lib.htp_b200_stream_status(dr.stream()) == 0


def test_parts_that_are_absent(pkg, lib):
    x = torch.randn((3, 500), device="cuda")
    out = torch.empty_like(x)
    empty = pkg.LogitsParams()
    assert lib.htp_b200_logits_process(out.data_ptr(), x.data_ptr(), 500, 3, 500, dr.ref(empty), dr.stream()) == 0
    assert torch.equal(out, x)
    mask = torch.full((3, 16), 0x55555555, dtype=torch.int32, device="cuda")
    only_mask = pkg.LogitsParams(mask=mask.data_ptr(), n_mask_rows=3)
    assert lib.htp_b200_logits_process(out.data_ptr(), x.data_ptr(), 500, 3, 500, dr.ref(only_mask), dr.stream()) == 0
    assert torch.equal(out[:, ::2], x[:, ::2]) and (out[:, 1::2] == -math.inf).all()
    hist, start = ints([4, 4, 9]), ints([0, 2, 2, 3])
    only_history = pkg.LogitsParams(history=hist.data_ptr(), history_start=start.data_ptr(), n_history=3)
    assert lib.htp_b200_logits_process(out.data_ptr(), x.data_ptr(), 500, 3, 500, dr.ref(only_history), dr.stream()) == 0
    assert torch.equal(out, x)


def test_bad_ranges_are_skipped_and_reported(pkg, lib):
    c = Case(pkg, 4, 3001, 40, 6, [0, -1, 0, -1], seed=5)
    want, size = c.want()
    assert lib.htp_b200_stream_status(dr.stream()) == 0
    for name, index, value, code, bad in (("history_start", 1, -4, 304, [0, 1]), ("history_start", 4, 10 ** 9, 304, [3]),
                                          ("bias_start", 2, 2 ** 31 - 1, 304, [1, 2]), ("mask_row", 0, 5, 305, [0]), ("mask_row", 2, -2, 305, [2])):
        t = c.buf[name]
        keep = t.clone()
        t[index] = value
        out = torch.full_like(c.x, 7.0)
        assert c.run(lib, out, c.x) == 0
        assert lib.htp_b200_stream_status(dr.stream()) == code
        good = [r for r in range(4) if r not in bad]
        close(out[good], want[good], size[good])
        t.copy_(keep)
