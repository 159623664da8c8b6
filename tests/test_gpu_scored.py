"""Decode, prefill and shared-prefix decode with changed scores against the
definition in 64 bits (oracle/scored_oracle.py, which derives the bounds)."""
import math

import pytest
import torch

from nanopd_amd import paged_kernels as pk
from oracle import scored_oracle as S

pytestmark = pytest.mark.gpu

BF16, F16 = torch.bfloat16, torch.float16


class Batch:
    """A fragmented pool and the tables of sequences of `lens` keys."""

    def __init__(self, device, lens, kvh, d, bs, dtype, fp8=False, seed=0, extra_cols=1):
        g = torch.Generator().manual_seed(seed)
        need = [-(-n // bs) for n in lens]
        total = sum(need) + 3
        order = torch.randperm(total, generator=g).to(torch.int32)
        self.table = torch.zeros(len(lens), max(need + [1]) + extra_cols, dtype=torch.int32)
        o = 0
        for i, n in enumerate(need):
            self.table[i, :n] = order[o:o + n]
            o += n
        kc = torch.randn(total, kvh, bs, d, generator=g)
        vc = torch.randn(total, kvh, bs, d, generator=g)
        self.ks = self.vs = None
        if fp8:
            self.ks = (0.03 + 0.05 * torch.rand(kvh, generator=g)).to(device)
            self.vs = (0.03 + 0.05 * torch.rand(kvh, generator=g)).to(device)
            self.kc = (kc * 12).clamp(-448, 448).to(torch.float8_e4m3fn).to(device)
            self.vc = (vc * 12).clamp(-448, 448).to(torch.float8_e4m3fn).to(device)
        else:
            self.kc, self.vc = kc.to(dtype).to(device), vc.to(dtype).to(device)
        self.table = self.table.to(device)
        self.lens, self.bs, self.d, self.dtype, self.device = lens, bs, d, dtype, device
        self.gen = g

    def seq_lens(self):
        return torch.tensor(self.lens, dtype=torch.int32, device=self.device)

    def queries(self, n, h, std=3.0):
        return (torch.randn(n, h, self.d, generator=self.gen) * std).to(self.dtype).to(self.device)

    def rows(self, s, n, table=None):
        t = self.table[s] if table is None else table
        k, v = S.gather(self.kc, t, n), S.gather(self.vc, t, n)
        if self.ks is not None:
            k = k.double() * self.ks.double()[None, :, None]
            v = v.double() * self.vs.double()[None, :, None]
        return k, v

    def kw(self):
        return {"k_scale": self.ks, "v_scale": self.vs}


def close(got, want, bound, what=""):
    assert torch.isfinite(got).all(), what
    over = (got.double() - want).abs() - bound(got.dtype)
    assert (over <= 0).all(), f"{what}: {float(over.max())} past the bound"


def check_decode(b, q, got, scale, softcap, slopes, window, first, prefix):
    for s, n in enumerate(b.lens):
        k, v = b.rows(s, n)
        want, bound = S.attend(q[s:s + 1], k, v, torch.tensor([n - 1]), n, scale, softcap, slopes,
                               window, None if first is None else first[s:s + 1],
                               0 if prefix is None else min(int(prefix[s]), n))
        close(got[s:s + 1], want, bound, f"sequence {s} of {n}")


DECODE = [
    # heads, kv heads, D, block, dtype, fp8, cap, slopes, window, masks, lens
    (12, 2, 128, 16, F16, False, 50.0, False, 0, False, [77]),
    (32, 8, 128, 16, BF16, False, 30.0, False, 0, False, [1, 15, 16, 17, 0, 300, 1025, 2500]),
    (32, 8, 128, 16, BF16, False, 0.0, True, 0, False, [1, 2, 260, 4000]),
    (8, 8, 128, 16, F16, False, 0.0, False, 100, True, [1, 99, 100, 101, 1000, 5000]),
    (64, 8, 128, 32, BF16, True, 20.0, True, 700, True, [5, 700, 701, 3001, 9000]),
    (34, 2, 64, 16, BF16, False, 40.0, False, 0, True, [3, 64, 1500]),
    (28, 4, 64, 8, F16, True, 0.0, True, 33, False, [3, 64, 1500]),
    (16, 8, 256, 16, BF16, False, 50.0, True, 0, False, [1, 18, 1100]),
    (16, 8, 256, 64, F16, True, 50.0, False, 500, True, [1, 18, 1100]),
    (10, 2, 96, 5, BF16, False, 25.0, False, 0, False, [4, 6, 333]),
    (6, 1, 40, 1, F16, False, 0.0, False, 7, True, [1, 7, 8, 50]),
    (32, 1, 32, 16, BF16, False, 1000.0, False, 0, False, [40, 900]),
    (4, 4, 248, 48, F16, False, 2e4, True, 0, False, [40, 300]),
    (5, 1, 160, 24, BF16, True, 0.0, False, 0, False, [40, 300]),
]


@pytest.mark.parametrize("case", DECODE, ids=range(len(DECODE)))
def test_decode(device, case):
    heads, kvh, d, bs, dtype, fp8, cap, slopes, window, masks, lens = case
    print("decode", case, flush=True)
    b = Batch(device, lens, kvh, d, bs, dtype, fp8, seed=heads + d)
    q = b.queries(len(lens), heads)
    sl = (2.0 ** (-8.0 * torch.arange(1, heads + 1) / heads)).to(device) if slopes else None
    first = prefix = None
    if masks:
        first = torch.tensor([n // 3 if i % 2 else 0 for i, n in enumerate(lens)], dtype=torch.int32,
                             device=device)
        prefix = torch.tensor([(5 * i) % 23 for i in range(len(lens))], dtype=torch.int32, device=device)
    out = torch.full_like(q, float("nan"))
    pk.paged_attention_scored(out, q, b.kc, b.vc, b.table, b.seq_lens(), d ** -0.5, bs,
                              b.table.size(1), softcap=cap, alibi_slopes=sl, window=window,
                              first_keys=first, prefix_lens=prefix, **b.kw())
    torch.cuda.synchronize()
    check_decode(b, q, out, d ** -0.5, cap, sl, window, first, prefix)


PREFILL = [
    # heads, kv heads, D, block, dtype, fp8, cap, slopes, window, docs, prefix, (chunk, before)s
    (12, 2, 128, 16, F16, False, 50.0, False, 0, 0, 0, [(1, 0), (33, 5)]),
    (32, 8, 128, 16, BF16, False, 30.0, False, 0, 0, 0, [(200, 700), (1, 64), (64, 0), (0, 9)]),
    (32, 8, 128, 16, BF16, False, 0.0, True, 0, 0, 0, [(130, 2000)]),
    (8, 8, 128, 16, F16, False, 0.0, False, 100, 0, 37, [(300, 0), (20, 1000)]),
    (16, 2, 128, 16, BF16, False, 0.0, False, 0, 40, 0, [(500, 30)]),
    (64, 8, 128, 32, BF16, True, 20.0, True, 300, 0, 70, [(90, 1200), (257, 0)]),
    (34, 2, 64, 16, BF16, False, 40.0, False, 0, 25, 0, [(150, 100)]),
    (28, 4, 64, 8, F16, True, 0.0, True, 33, 0, 0, [(65, 64)]),
    (16, 8, 256, 16, BF16, False, 50.0, True, 0, 0, 500, [(140, 200)]),
    (16, 8, 256, 64, F16, True, 50.0, False, 128, 30, 20, [(140, 200), (3, 1000)]),
    (10, 2, 96, 5, BF16, False, 25.0, False, 0, 0, 0, [(77, 8)]),
    (6, 1, 40, 1, F16, False, 0.0, False, 7, 0, 3, [(90, 0)]),
    (4, 4, 248, 48, F16, False, 2e4, True, 0, 0, 0, [(40, 300)]),
    (5, 1, 160, 24, BF16, True, 1000.0, False, 0, 0, 0, [(40, 300)]),
    (4, 2, 32, 16, BF16, False, 0.0, False, 0, 0, 0, [(700, 0), (5, 0)]),
]


def masks_of(chunks, docs, prefix, device):
    """first_keys (documents of `docs` tokens) and prefix_lens."""
    first = pre = None
    if docs:
        first = torch.cat([(torch.arange(c, c + q) // docs * docs) for q, c in chunks]).to(torch.int32)
        first = first.to(device)
    if prefix:
        pre = torch.tensor([prefix + 3 * i for i in range(len(chunks))], dtype=torch.int32, device=device)
    return first, pre


def check_prefill(b, q, got, chunks, scale, cap, sl, window, first, pre):
    o = 0
    for s, (n, c) in enumerate(chunks):
        if n == 0:
            continue
        k, v = b.rows(s, c + n)
        want, bound = S.attend(q[o:o + n], k, v, torch.arange(c, c + n), c + n, scale, cap, sl, window,
                               None if first is None else first[o:o + n],
                               0 if pre is None else min(int(pre[s]), c + n))
        close(got[o:o + n], want, bound, f"sequence {s}: {n} on {c}")
        o += n


@pytest.mark.parametrize("case", PREFILL, ids=range(len(PREFILL)))
def test_prefill(device, case):
    heads, kvh, d, bs, dtype, fp8, cap, slopes, window, docs, prefix, chunks = case
    print("prefill", case, flush=True)
    b = Batch(device, [q + c for q, c in chunks], kvh, d, bs, dtype, fp8, seed=heads + d)
    total = sum(q for q, _ in chunks)
    q = b.queries(total + 3, heads)
    sl = (2.0 ** (-8.0 * torch.arange(1, heads + 1) / heads)).to(device) if slopes else None
    first, pre = masks_of(chunks, docs, prefix, device)
    if first is not None:
        first = torch.cat([first, first.new_zeros(3)])
    cu = torch.tensor([0] + [q for q, _ in chunks], device=device).cumsum(0).to(torch.int32)
    out = torch.full_like(q, 7.0)
    pk.paged_prefill_attention_scored(out, q, b.kc, b.vc, b.table, cu, b.seq_lens(), d ** -0.5, bs,
                                      b.table.size(1), max(n for n, _ in chunks), softcap=cap,
                                      alibi_slopes=sl, window=window, first_keys=first,
                                      prefix_lens=pre, **b.kw())
    torch.cuda.synchronize()
    assert (out[total:] == 7.0).all()      # rows past the last sequence
    check_prefill(b, q, out[:total], chunks, d ** -0.5, cap, sl, window, first, pre)


SHARED = [
    # heads, kv heads, D, block, dtype, fp8, cap, slopes, window, [(shared, [own...])...]
    (12, 2, 128, 16, F16, False, 0.0, False, 0, [(512, [1, 20, 60, 33])]),
    (32, 8, 128, 16, BF16, False, 50.0, False, 0, [(2048, [1, 500, 0, 17, 300] * 8)]),
    (64, 8, 128, 16, BF16, True, 30.0, False, 0, [(640, [3, 9]), (0, [40]), (1600, [100] * 5)]),
    (8, 8, 64, 32, F16, False, 0.0, True, 0, [(320, [5] * 3), (64, [700])]),
    (16, 8, 256, 16, BF16, False, 0.0, False, 300, [(1024, [5, 290, 310, 900])]),
    (10, 2, 96, 8, BF16, False, 20.0, True, 0, [(80, [0, 1])]),
    (34, 2, 64, 16, BF16, True, 0.0, False, 0, [(160, [4] * 11)]),
]


@pytest.mark.parametrize("case", SHARED, ids=range(len(SHARED)))
def test_shared(device, case):
    heads, kvh, d, bs, dtype, fp8, cap, slopes, window, groups = case
    print("shared", case, flush=True)
    lens = [sh + own for sh, owns in groups for own in owns]
    b = Batch(device, lens, kvh, d, bs, dtype, fp8, seed=heads + d)
    cu, i = [0], 0
    for sh, owns in groups:
        for k in range(1, len(owns)):
            b.table[i + k, :sh // bs] = b.table[i, :sh // bs]
        i += len(owns)
        cu.append(i)
    q = b.queries(len(lens), heads)
    sl = (2.0 ** (-8.0 * torch.arange(1, heads + 1) / heads)).to(device) if slopes else None
    out = torch.full_like(q, float("nan"))
    pk.paged_attention_shared(out, q, b.kc, b.vc, b.table, b.seq_lens(), d ** -0.5, bs,
                              b.table.size(1), torch.tensor(cu, dtype=torch.int32, device=device),
                              torch.tensor([g[0] for g in groups], dtype=torch.int32, device=device),
                              max(g[0] for g in groups), softcap=cap, alibi_slopes=sl, window=window,
                              **b.kw())
    torch.cuda.synchronize()
    check_decode(b, q, out, d ** -0.5, cap, sl, window, None, None)


U = {BF16: 2.0 ** -8, F16: 2.0 ** -11}


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("rows,width", [(1, 8), (3, 520), (7, 1536), (5, 2048), (37, 2056), (527, 4096),
                                        (9, 5120), (2, 8192), (3, 8200), (3, 100), (0, 64)])
@pytest.mark.parametrize("gate", ["none", "column", "row", "full", "strided"])
def test_block_norms(device, dtype, rows, width, gate):
    """x within one rounding of 64 bits (a few fp32 ones besides), h within one
    of what the stored x gives."""
    print("block_norms", dtype, rows, width, gate, flush=True)
    g = torch.Generator(device=device).manual_seed(rows + width)
    rnd = lambda *s: torch.randn(*s, generator=g, device=device)
    x, delta = (rnd(rows, width) * 4).to(dtype), rnd(rows, width).to(dtype)
    post, w = (1 + 0.2 * rnd(width)).to(dtype), (1 + 0.2 * rnd(width)).to(dtype)
    gt = {"none": None, "column": rnd(width), "row": rnd(rows, 1), "full": rnd(rows, width),
          "strided": rnd(rows, width + 16)[:, 8:width + 8]}[gate]
    gt = None if gt is None else gt.to(dtype)
    if gate == "strided":
        wide = torch.zeros(rows, width + 16, dtype=dtype, device=device)
        wide[:, 8:width + 8] = gt
        gt = wide[:, 8:width + 8]
    xd, dd = x.double(), delta.double()
    d64 = dd * torch.rsqrt(dd.pow(2).mean(-1, keepdim=True) + 1e-6) * post.double()
    if gt is not None:
        d64 = gt.double() * d64
    want = 0.7 * xd + d64
    h = pk.block_norms(x, delta, post, w, 1e-6, gate=gt, residual_scale=0.7)
    # fp32 roundings: (width / 64 + 8) additions of the statistic at most, a few
    # products; fp16 also rounds below its normal range
    e32 = 2.0 ** -24 * (width / 64 + 16)
    tiny = 2.0 ** -25 if dtype == F16 else 0.0
    assert ((x.double() - want).abs() <= U[dtype] * want.abs() * 1.001 + tiny
            + e32 * (0.7 * xd.abs() + d64.abs())).all()
    f = x.double()
    wh = f * torch.rsqrt(f.pow(2).mean(-1, keepdim=True) + 1e-6) * w.double()
    assert ((h.double() - wh).abs() <= (U[dtype] * 1.001 + e32) * wh.abs() + tiny).all()
