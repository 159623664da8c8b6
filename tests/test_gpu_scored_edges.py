"""Scored attention and block norms where they can go wrong: keys that must not be
read for anything, strides, streams, graphs, workspaces, groups of every kind, and
a model that uses all of them together."""
import pytest
import torch

from nanopd_amd import paged_kernels as pk
from nanopd_amd.graphs import DecodeGraphs
from nanopd_amd.qwen3 import PagedQwen3, Qwen3Config, StepBatch
from oracle import scored_oracle as S
from .test_gpu_scored import BF16, F16, Batch, check_decode, check_prefill, close

pytestmark = pytest.mark.gpu


def cu_of(counts, device):
    return torch.tensor([0] + counts, device=device).cumsum(0).to(torch.int32)


def poison(b, keep, value):
    """Every pool row that is not kept (sequence -> keys) becomes `value`."""
    mask = torch.ones(b.kc.size(0), b.bs, dtype=torch.bool)
    for s, keys in keep.items():
        for j in keys:
            mask[int(b.table[s, j // b.bs]), j % b.bs] = False
    mask = mask.to(b.device)
    for c in (b.kc, b.vc):
        if b.ks is not None:
            raw = c.view(torch.uint8)
            raw.copy_(torch.where(mask[:, None, :, None], torch.full_like(raw, 0x7f), raw))
        else:
            c.copy_(torch.where(mask[:, None, :, None], torch.full_like(c, value), c))


VALUES = [float("nan"), float("inf"), -float("inf")]


@pytest.mark.parametrize("value", VALUES)
@pytest.mark.parametrize("d,bs,fp8,dtype", [(128, 16, False, BF16), (64, 5, False, F16), (256, 32, True, BF16)])
def test_unseen_keys_have_no_effect_on_decode(device, value, d, bs, fp8, dtype):
    lens, window, first, pre = [1, 40, 333, 90], 30, [0, 0, 2, 85], [0, 7, 5, 88]
    b = Batch(device, lens, 2, d, bs, dtype, fp8, seed=3)
    q = b.queries(4, 8)
    keep = {s: [j for j in range(n) if j >= f and (n - 1 - j < window or j < p)]
            for s, (n, f, p) in enumerate(zip(lens, first, pre))}
    f, p = (torch.tensor(x, dtype=torch.int32, device=device) for x in (first, pre))
    poison(b, keep, value)
    out = torch.empty_like(q)
    pk.paged_attention_scored(out, q, b.kc, b.vc, b.table, b.seq_lens(), d ** -0.5, bs, b.table.size(1),
                              softcap=20.0, window=window, first_keys=f, prefix_lens=p, **b.kw())
    for s, n in enumerate(lens):
        k, v = b.rows(s, n)
        sel = torch.tensor(keep[s], device=device)
        k, v = (torch.zeros_like(x).index_copy_(0, sel, x[sel]) for x in (k, v))
        want, bound = S.attend(q[s:s + 1], k, v, torch.tensor([n - 1]), n, d ** -0.5, 20.0, None, window,
                               f[s:s + 1], min(pre[s], n))
        close(out[s:s + 1], want, bound, f"sequence {s}")


@pytest.mark.parametrize("value", VALUES)
@pytest.mark.parametrize("d,bs,fp8,dtype", [(128, 16, False, BF16), (64, 5, False, F16), (256, 32, True, BF16)])
def test_unseen_keys_have_no_effect_on_chunks(device, value, d, bs, fp8, dtype):
    """A row's own future holds keys that later rows see: theirs is the poison, kept
    out of one document by the other and out of windows."""
    chunks, window = [(70, 90), (33, 0)], 40
    b = Batch(device, [q + c for q, c in chunks], 2, d, bs, dtype, fp8, seed=4)
    q = b.queries(103, 8)
    first = torch.cat([torch.full((70,), 60), torch.zeros(33)]).to(torch.int32).to(device)
    # keys 0 .. 59 of sequence 0 are before every row's document
    poison(b, {0: range(60, 160), 1: range(33)}, value)
    # and one row of sequence 1 is the poison of all rows before it
    bad = int(b.table[1, 20 // bs])
    raw = b.vc.view(torch.uint8) if fp8 else b.vc
    raw[bad, :, 20 % bs] = 0x7f if fp8 else value
    out = torch.empty_like(q)
    pk.paged_prefill_attention_scored(out, q, b.kc, b.vc, b.table, cu_of([70, 33], device), b.seq_lens(),
                                      d ** -0.5, bs, b.table.size(1), 70, softcap=20.0, window=window,
                                      first_keys=first, **b.kw())
    for s, (lo, n, c) in enumerate([(0, 70, 90), (70, 20, 0)]):   # the rows that do not see the bad key
        k, v = b.rows(s, c + n)
        k, v = (torch.where(torch.arange(c + n, device=device)[:, None, None] < (60 if s == 0 else 0),
                            torch.zeros_like(x), x) for x in (k, v))
        want, bound = S.attend(q[lo:lo + n], k, v, torch.arange(c, c + n), c + n, d ** -0.5, 20.0, None,
                               window, first[lo:lo + n])
        close(out[lo:lo + n], want, bound, f"sequence {s}")
    assert not torch.isfinite(out[90:103]).any()   # those that do


@pytest.mark.parametrize("value", VALUES)
def test_unseen_keys_have_no_effect_on_shared(device, value):
    lens = [70, 100, 65]
    b = Batch(device, lens, 2, 128, 16, BF16, seed=5)
    b.table[1:, :4] = b.table[0, :4]
    q = b.queries(3, 8)
    poison(b, {s: range(n) for s, n in enumerate(lens)}, value)
    out = torch.empty_like(q)
    pk.paged_attention_shared(out, q, b.kc, b.vc, b.table, b.seq_lens(), 0.1, 16, b.table.size(1),
                              cu_of([3], device), torch.tensor([64], dtype=torch.int32, device=device), 64)
    check_decode(b, q, out, 0.1, 0.0, None, 0, None, None)


def test_lowest_and_infinite_scores(device):
    """Scores past the cap on either side, and a distance term that leaves one key."""
    b = Batch(device, [50, 300], 1, 64, 16, F16, seed=6)
    q = b.queries(2, 4, std=200.0)
    sl = torch.tensor([0.0, 1.0, 500.0, 60000.0], device=device)
    for cap in (0.0, 5.0):
        out = torch.empty_like(q)
        pk.paged_attention_scored(out, q, b.kc, b.vc, b.table, b.seq_lens(), 1.0, 16, b.table.size(1),
                                  softcap=cap, alibi_slopes=sl)
        check_decode(b, q, out, 1.0, cap, sl, 0, None, None)


# -- strides, streams, empties --------------------------------------------------------

def test_strided_queries_and_outputs(device):
    b = Batch(device, [30, 77, 500], 2, 64, 16, BF16, seed=7)
    wide = b.queries(3, 24)                       # 8 heads of a fused projection's 24
    q = wide[:, 8:16]
    buf = torch.full((3, 12, 64), 7.0, dtype=BF16, device=device)
    out = buf[:, 2:10]
    pk.paged_attention_scored(out, q, b.kc, b.vc, b.table, b.seq_lens(), 0.125, 16, b.table.size(1),
                              softcap=30.0)
    check_decode(b, q, out, 0.125, 30.0, None, 0, None, None)
    assert (buf[:, :2] == 7.0).all() and (buf[:, 10:] == 7.0).all()
    chunks = [(30, 0), (7, 70), (90, 410)]
    wide = b.queries(127, 24)
    q = wide[:, 8:16]
    buf = torch.full((127, 12, 64), 7.0, dtype=BF16, device=device)
    out = buf[:, 2:10]
    pk.paged_prefill_attention_scored(out, q, b.kc, b.vc, b.table, cu_of([30, 7, 90], device),
                                      b.seq_lens(), 0.125, 16, b.table.size(1), 90, softcap=30.0)
    check_prefill(b, q, out, chunks, 0.125, 30.0, None, 0, None, None)
    assert (buf[:, :2] == 7.0).all() and (buf[:, 10:] == 7.0).all()


def test_rows_of_a_stride_past_32_bits(device):
    """Token stride of 2^30 elements: row 2 lies 2^32 bytes into the buffers."""
    b = Batch(device, [20, 33, 40], 1, 32, 16, BF16, seed=8)
    n = 2 * 2 ** 30 + 4 * 32
    qb, ob = (torch.empty(n, dtype=BF16, device=device) for _ in range(2))
    q, out = (x.as_strided((3, 4, 32), (2 ** 30, 32, 1)) for x in (qb, ob))
    q.copy_(b.queries(3, 4))
    pk.paged_attention_scored(out, q, b.kc, b.vc, b.table, b.seq_lens(), 0.2, 16, b.table.size(1))
    check_decode(b, q, out, 0.2, 0.0, None, 0, None, None)
    out.zero_()
    pk.paged_prefill_attention_scored(out, q, b.kc, b.vc, b.table, cu_of([1, 1, 1], device), b.seq_lens(),
                                      0.2, 16, b.table.size(1), 1)
    check_decode(b, q, out, 0.2, 0.0, None, 0, None, None)


def test_pool_past_32_bits(device):
    """A pool of 5 GB per cache whose last blocks hold the sequence."""
    nb = 5 * 2 ** 30 // (16 * 128 * 2)
    kc, vc = (torch.empty(nb, 1, 16, 128, dtype=BF16, device=device) for _ in range(2))
    b = Batch(device, [100], 1, 128, 16, BF16, seed=9)
    for big, small in ((kc, b.kc), (vc, b.vc)):
        big[nb - small.size(0):].copy_(small)
    table = b.table + (nb - b.kc.size(0))
    q = b.queries(1, 8)
    out = torch.empty_like(q)
    pk.paged_attention_scored(out, q, kc, vc, table, b.seq_lens(), 0.1, 16, table.size(1))
    check_decode(b, q, out, 0.1, 0.0, None, 0, None, None)
    q = b.queries(40, 8)
    out = torch.empty_like(q)
    pk.paged_prefill_attention_scored(out, q, kc, vc, table, cu_of([40], device), b.seq_lens(), 0.1, 16,
                                      table.size(1), 40)
    check_prefill(b, q, out, [(40, 60)], 0.1, 0.0, None, 0, None, None)


def test_other_stream_and_empty_calls(device):
    b = Batch(device, [300, 9], 2, 128, 16, BF16, seed=10)
    q = b.queries(2, 8)
    out = torch.empty_like(q)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        pk.paged_attention_scored(out, q, b.kc, b.vc, b.table, b.seq_lens(), 0.1, 16, b.table.size(1))
    torch.cuda.current_stream().wait_stream(side)
    check_decode(b, q, out, 0.1, 0.0, None, 0, None, None)
    e = q[:0]
    pk.paged_attention_scored(e, e, b.kc, b.vc, b.table, b.seq_lens(), 0.1, 16, b.table.size(1))
    pk.paged_prefill_attention_scored(e, e, b.kc, b.vc, b.table, cu_of([0, 0], device), b.seq_lens(), 0.1,
                                      16, b.table.size(1), 1)
    # no chunk has a token: nothing is written
    out.fill_(7.0)
    pk.paged_prefill_attention_scored(out, q, b.kc, b.vc, b.table, cu_of([0, 0], device), b.seq_lens(), 0.1,
                                      16, b.table.size(1), 1)
    torch.cuda.synchronize()
    assert (out == 7.0).all()


# -- workspaces and graphs ---------------------------------------------------------------

def all_ops(b, q, qc, cu, groups, outs, ws=(None, None, None)):
    n = b.table.size(1)
    pk.paged_attention_scored(outs[0], q, b.kc, b.vc, b.table, b.seq_lens_d, 0.1, 16, n, softcap=30.0,
                              workspace=ws[0])
    pk.paged_attention_shared(outs[1], q, b.kc, b.vc, b.table, b.seq_lens_d, 0.1, 16, n, *groups,
                              softcap=30.0, workspace=ws[1])
    pk.paged_prefill_attention_scored(outs[2], qc, b.kc, b.vc, b.table, cu, b.seq_lens_d, 0.1, 16, n,
                                      max_q_len=300, softcap=30.0, workspace=ws[2])


def graph_batch(device):
    lens = [1200, 1100, 1099, 900]
    b = Batch(device, lens, 2, 128, 16, BF16, seed=11)
    b.table[1:, :50] = b.table[0, :50]
    b.seq_lens_d = b.seq_lens()
    counts = [300, 1, 64, 129]
    groups = (cu_of([4], device), torch.tensor([800], dtype=torch.int32, device=device), 800)
    q, qc = b.queries(4, 16), b.queries(sum(counts), 16)
    return b, q, qc, cu_of(counts, device), groups, counts


def check_all(b, q, qc, counts, outs):
    check_decode(b, q, outs[0], 0.1, 30.0, None, 0, None, None)
    check_decode(b, q, outs[1], 0.1, 30.0, None, 0, None, None)
    check_prefill(b, qc, outs[2], [(n, m - n) for n, m in zip(counts, b.lens)], 0.1, 30.0, None, 0, None, None)


def test_one_workspace_serves_every_call(device):
    """Dirty, shared by the three ops one after another, and with a guard behind it."""
    b, q, qc, cu, groups, counts = graph_batch(device)
    n = b.table.size(1)
    need = [pk.scored_workspace_bytes(4, 16, 2, 128, 16, n),
            pk.shared_workspace_bytes(4, 16, 2, 128, 16, n, 1, 800),
            pk.prefill_scored_workspace_bytes(4, sum(counts), 16, 2, 128, 300, n * 16)]
    assert min(need) > 0
    buf = torch.full((max(need) + 4096,), 0xff, dtype=torch.uint8, device=device)
    for _ in range(2):
        outs = [torch.empty_like(x) for x in (q, q, qc)]
        all_ops(b, q, qc, cu, groups, outs, [buf[:k] for k in need])
        check_all(b, q, qc, counts, outs)
    assert (buf[max(need):] == 0xff).all()
    for i in range(3):
        ws = [buf[:k] for k in need]
        ws[i] = buf[:need[i] - 1]
        with pytest.raises(RuntimeError):
            all_ops(b, q, qc, cu, groups, outs, ws)


@pytest.mark.parametrize("explicit", [False, True])
def test_graphs_replay(device, explicit):
    """Two graphs (with one explicit workspace between them, or one each) replayed in
    turn, between eager calls and synchronisations, with inputs that change."""
    b, q, qc, cu, groups, counts = graph_batch(device)
    ws = (None, None, None)
    if explicit:
        buf = torch.full((1 << 28,), 0xff, dtype=torch.uint8, device=device)
        ws = (buf, buf, buf)
    x, delta = qc.view(len(qc), -1), torch.randn_like(qc.view(len(qc), -1))
    w = torch.rand(x.size(1), device=device).to(BF16)
    outs = [[torch.zeros_like(t) for t in (q, q, qc, x, x)] for _ in range(2)]

    def run(o):
        all_ops(b, q, qc, cu, groups, o, ws)
        o[4].copy_(pk.block_norms(o[2].view(len(qc), -1), delta, w, w, 1e-6, gate=w, x_out=o[3]))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run(outs[0])
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graphs = []
    for o in outs:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            run(o)
        graphs.append(g)
    for turn in range(4):
        q.copy_(b.queries(4, 16))
        qc.copy_(b.queries(len(qc), 16))
        eager = [torch.zeros_like(t) for t in outs[0]]
        run(eager)
        if turn % 2:
            torch.cuda.synchronize()
        for g, o in zip(graphs, outs):
            g.replay()
            for a, e in zip(o, eager):
                assert torch.equal(a, e)
    check_all(b, q, qc, counts, outs[1])


def test_results_repeat_bit_for_bit(device):
    """No atomics: two calls, also side by side on two streams, give the same bits."""
    b, q, qc, cu, groups, counts = graph_batch(device)
    first = [torch.empty_like(x) for x in (q, q, qc)]
    all_ops(b, q, qc, cu, groups, first)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = [[torch.empty_like(x) for x in (q, q, qc)] for _ in streams]
    torch.cuda.synchronize()
    for _ in range(3):
        for s, o in zip(streams, outs):
            with torch.cuda.stream(s):
                all_ops(b, q, qc, cu, groups, o)
    torch.cuda.synchronize()
    for o in outs:
        assert all(torch.equal(x, y) for x, y in zip(o, first))


@pytest.mark.parametrize("lens", [
    [400 + (37 * i) % 90 for i in range(700)],               # more than are counted, even
    [(131 * i) % 1500 for i in range(600)],                  # ragged
    [0] * 5 + [3000] + [1] * 9, [0] * 8, [5000], [257, 256, 255, 64, 65],
], ids=range(6))
def test_parts_of_many_lengths(device, lens):
    b = Batch(device, lens, 1, 64, 16, F16, seed=21)
    q = b.queries(len(lens), 4)
    out = torch.full_like(q, float("nan"))
    pk.paged_attention_scored(out, q, b.kc, b.vc, b.table, b.seq_lens(), 0.1, 16, b.table.size(1),
                              softcap=15.0)
    check_decode(b, q, out, 0.1, 15.0, None, 0, None, None)


# -- groups ---------------------------------------------------------------------------------

def shared_case(device, lens, groups, kvh=2, heads=8, d=64, seed=12, max_shared=None, tables=None):
    """groups: (first, last + 1, shared keys)."""
    b = Batch(device, lens, kvh, d, 16, BF16, seed=seed)
    for lo, hi, sh in (g for g in groups if g[1] > g[0]):
        b.table[lo:hi, : -(-sh // 16)] = b.table[lo, : -(-sh // 16)].clone()
    q = b.queries(len(lens), heads)
    cu = torch.tensor([g[0] for g in groups] + [groups[-1][1]], dtype=torch.int32, device=device)
    sh = torch.tensor([g[2] for g in groups], dtype=torch.int32, device=device)
    out = torch.full_like(q, float("nan"))
    pk.paged_attention_shared(out, q, b.kc, b.vc, b.table, b.seq_lens(), d ** -0.5, 16, b.table.size(1), cu,
                              sh, int(sh.max()) if max_shared is None else max_shared, softcap=25.0)
    check_decode(b, q, out, d ** -0.5, 25.0, None, 0, None, None)


@pytest.mark.parametrize("lens,groups,max_shared", [
    ([100, 200, 300], [(1, 3, 96)], None),                       # a sequence before every group
    ([100, 200, 300, 50], [(0, 2, 96)], None),                   # and behind
    ([100, 200], [(0, 0, 64), (0, 2, 96), (2, 2, 32)], None),    # groups without a sequence
    ([40, 0, 200, 96, 95], [(0, 5, 96)], None),                  # shorter than the shared keys, empty
    ([300, 300], [(0, 2, 288)], 100),                            # shared keys past the bound: per sequence
    ([300, 300], [(0, 2, 288)], 0),
    ([33, 34], [(0, 2, 17)], None),                              # no whole block shared
    ([500], [(0, 1, 500)], None),                                # a group of one, all of it shared
])
def test_groups(device, lens, groups, max_shared):
    shared_case(device, lens, groups, max_shared=max_shared)


def test_many_groups(device):
    """More groups than a list has entries, some without shared keys."""
    lens = [20 + (7 * i) % 60 for i in range(1200)]
    groups = [(2 * i, 2 * i + 2, [16, 0, 19, 16][i % 4]) for i in range(600)]
    shared_case(device, lens, groups, kvh=1, heads=2, d=32)


def test_large_group(device):
    """Tiles of many sequences, one prefix longer than a list of blocks."""
    shared_case(device, [9000 + i % 5 for i in range(150)], [(0, 150, 8992)], heads=16)


def test_lists_that_do_not_ascend_stay_in_bounds(device):
    """Groups that overlap or run backwards have no defined result for their own
    sequences; nothing outside out's rows is touched and the call ends."""
    b = Batch(device, [400] * 6, 2, 64, 16, BF16, seed=13)
    b.table[1:, :20] = b.table[0, :20]
    q = b.queries(6, 8)
    buf = torch.full((8, 8, 64), 7.0, dtype=BF16, device=device)
    for cu in ([4, 2, 0], [0, 6, 3, 6], [0, 100, -5, 6], [5, 5, 5]):
        sh = torch.full((len(cu) - 1,), 320, dtype=torch.int32, device=device)
        pk.paged_attention_shared(buf[1:7], q, b.kc, b.vc, b.table, b.seq_lens(), 0.1, 16, b.table.size(1),
                                  torch.tensor(cu, dtype=torch.int32, device=device), sh, 320)
        torch.cuda.synchronize()
    assert (buf[0] == 7.0).all() and (buf[7] == 7.0).all()


def test_same_block_twice_and_bad_pages(device):
    """A table may name a block more than once; ids outside the pool are clamped."""
    b = Batch(device, [64, 48], 2, 64, 16, BF16, seed=14)
    b.table[0, 2] = b.table[0, 1]
    b.table[1, :3] = b.table[0, 1]
    q = b.queries(2, 8)
    out = torch.empty_like(q)
    pk.paged_attention_scored(out, q, b.kc, b.vc, b.table, b.seq_lens(), 0.1, 16, b.table.size(1))
    check_decode(b, q, out, 0.1, 0.0, None, 0, None, None)
    wild = b.table.clone()
    wild[0, 0], wild[1, 1] = -5, 10 ** 9
    clamped = b.table.clone()
    clamped[0, 0], clamped[1, 1] = 0, b.kc.size(0) - 1
    outs = [torch.empty_like(q) for _ in range(2)]
    for o, t in zip(outs, (wild, clamped)):
        pk.paged_attention_scored(o, q, b.kc, b.vc, t, b.seq_lens(), 0.1, 16, t.size(1))
    assert torch.equal(*outs)


@pytest.mark.parametrize("d,heads", [(64, 8), (128, 8), (256, 4)])
def test_chunks_of_every_count(device, d, heads):
    """From one tile (one workgroup) over shares of tiles to whole tiles."""
    for chunks in ([(1, 0)], [(40, 3000)], [(260, 10)] * 5, [(70, 900)] * 40, [(2, 3)] * 600):
        print(d, chunks[0], len(chunks), flush=True)
        b = Batch(device, [q + c for q, c in chunks], heads // 4, d, 16, F16, seed=15)
        q = b.queries(sum(n for n, _ in chunks), heads)
        out = torch.full_like(q, float("nan"))
        pk.paged_prefill_attention_scored(out, q, b.kc, b.vc, b.table, cu_of([n for n, _ in chunks], device),
                                          b.seq_lens(), d ** -0.5, 16, b.table.size(1),
                                          max(n for n, _ in chunks), softcap=40.0)
        assert torch.isfinite(out).all()
        some = chunks[:3]
        n = sum(x for x, _ in some)
        check_prefill(b, q[:n], out[:n], some, d ** -0.5, 40.0, None, 0, None, None)


def test_padded_buffers(device):
    """A batch in a much longer buffer, whose rows past the last sequence stay, and
    sequences without a token between others."""
    b = Batch(device, [700, 90, 33], 2, 64, 16, BF16, seed=20)
    n = 40000
    q = torch.zeros(n, 8, 64, dtype=BF16, device=device)
    q[:150] = b.queries(150, 8)
    out = torch.full_like(q, 7.0)
    pk.paged_prefill_attention_scored(out, q, b.kc, b.vc, b.table, cu_of([100, 50, 0], device),
                                      b.seq_lens(), 0.1, 16, b.table.size(1), 100, softcap=9.0)
    check_prefill(b, q[:150], out[:150], [(100, 600), (50, 40), (0, 33)], 0.1, 9.0, None, 0, None, None)
    assert (out[150:] == 7.0).all()


def test_max_context_len_bounds_only_the_plan(device):
    b = Batch(device, [700, 90], 2, 64, 16, BF16, seed=16)
    q = b.queries(150, 8)
    for bound in (1, 700, 4000):
        out = torch.empty_like(q)
        pk.paged_prefill_attention_scored(out, q, b.kc, b.vc, b.table, cu_of([100, 50], device), b.seq_lens(),
                                          0.1, 16, b.table.size(1), 100, bound)
        check_prefill(b, q, out, [(100, 600), (50, 40)], 0.1, 0.0, None, 0, None, None)


# -- block norms ------------------------------------------------------------------------------

def test_block_norms_writes_where_it_reads(device):
    g = torch.Generator(device=device).manual_seed(17)
    x, d, gate = (torch.randn(37, 520, device=device, generator=g).to(BF16) for _ in range(3))
    w = torch.rand(520, device=device, generator=g).to(BF16)
    keep = torch.empty_like(x)
    h = pk.block_norms(x, d, w, w, 1e-6, gate=gate, residual_scale=0.5, x_out=keep)
    for which in ("x", "delta", "gate"):
        t = {"x": x.clone(), "delta": d.clone(), "gate": gate.clone()}
        h2 = pk.block_norms(t["x"], t["delta"], w, w, 1e-6, gate=t["gate"], residual_scale=0.5,
                            x_out=t[which])
        assert torch.equal(h2, h) and torch.equal(t[which], keep)


# -- together, in a model ----------------------------------------------------------------------

CFG = Qwen3Config(num_layers=2, hidden=256, num_heads=8, num_kv_heads=2, head_dim=64, intermediate=512,
                  vocab=1000, init_std=0.05, attn_softcap=20.0, window=200, block_norms=True)


def plain_attention(cfg, scale):
    """The definition in 64 bits in place of the kernels."""
    def attend(layer, q, kc, vc, b, out):
        m = b.meta
        cu, sl = m.cu_seqlens_q.tolist(), m.seq_lens.tolist()
        for s, n in enumerate(sl):
            a, e = cu[s], cu[s + 1]
            k, v = S.gather(kc, m.block_tables[s], n), S.gather(vc, m.block_tables[s], n)
            o, _ = S.attend(q[a:e], k, v, torch.arange(n - (e - a), n), n, scale, cfg.attn_softcap, None,
                            cfg.window)
            out[a:e] = o.to(out.dtype)
    return attend


def model_batch(device, seqs, npf, shared=None):
    g = torch.Generator().manual_seed(19)
    total = sum(n for n, _, _ in seqs)
    tp = sum(n for n, _, _ in seqs[:npf])
    meta = pk.pack_metadata(seqs, 16, device)
    return StepBatch(torch.randint(0, CFG.vocab, (total,), generator=g).to(device), meta, npf, tp, None,
                     max([n for n, _, _ in seqs[:npf]] + [0]), shared=shared)


def test_model_with_scored_attention_and_block_norms(device):
    """A prefill step, a mixed step and a decode step over a forked prefix, against
    the same model with the definition in the place of the attention kernels and
    torch operations in that of block_norms."""
    hip = PagedQwen3(CFG, 128, 16, device, seed=1)
    ref = PagedQwen3(CFG, 128, 16, device, seed=1, attention=plain_attention(CFG, hip.scale))
    t0, t1 = list(range(20)), list(range(20, 36))
    forks = [t0[:15] + [40 + i, 50 + i] for i in range(4)]
    steps = [model_batch(device, [(240, 0, t0), (100, 0, t1)], 2),
             model_batch(device, [(60, 100, t1)] + [(1, 240, f) for f in forks], 1)]
    last = [(1, 241, f) for f in forks] + [(1, 160, t1)]
    sh = pk.find_shared_prefixes([t for _, _, t in last], [c + 1 for _, c, _ in last], 16, device)
    assert sh.cu_groups.tolist() == [0, 4, 5] and sh.shared_lens.tolist() == [240, 0]
    steps.append(model_batch(device, last, 0, sh))
    for i, b in enumerate(steps):
        got = hip.forward(b)
        if i == 2:
            # the shared form against the one without, before its own comparison
            plain = hip.forward(model_batch(device, last, 0))
            assert (got - plain).abs().max() <= 2e-2 * plain.abs().max()
        want = ref.forward(b)
        # hidden values pass a handful of bf16 roundings (2^-8 each) per layer, two layers
        err, spread = (got - want).abs().max().item(), want.abs().max().item()
        print(f"step {i}: logits off by {err:.3e} of {spread:.2f}", flush=True)
        assert err <= 10 * 2.0 ** -8 * spread


def test_model_options_are_off_by_default(device):
    """Without options no scored op runs, and results are those of the plain layer."""
    cfg = Qwen3Config(**{**CFG.__dict__, "attn_softcap": 0.0, "window": 0, "block_norms": False})
    m = PagedQwen3(cfg, 64, 16, device, seed=1)
    assert m.layers[0]["attn_out_norm"] is None
    with pytest.raises(ValueError):
        PagedQwen3(CFG, 64, 16, device, seed=1).load_hf_state_dict({})
    b = model_batch(device, [(50, 0, [0, 1, 2, 3]), (1, 20, [8, 9])], 1)
    names = []
    keep = pk._call_on
    try:
        pk._call_on = lambda dev, name, *a: (names.append(name), keep(dev, name, *a))[1]
        m.forward(b)
    finally:
        pk._call_on = keep
    assert names == []


@pytest.mark.parametrize("kv", ["auto", "fp8"])
def test_decode_graphs_of_such_a_model(device, kv):
    """The engine's captured decode steps against eager ones, padded batches too."""
    m = PagedQwen3(CFG, 128, 16, device, seed=2, kv_cache_dtype=kv)
    tables = [list(range(0, 20)), list(range(20, 40)), list(range(40, 60))]
    lens = [250, 31, 7]
    m.forward(model_batch(device, [(n, 0, t) for n, t in zip(lens, tables)], 3))
    graphs = DecodeGraphs(m, max_width=32)
    for turn in range(3):
        ids = [5 + turn, 17, 900]
        pos = [n + turn for n in lens]
        b = model_batch(device, [(1, p, t) for p, t in zip(pos, tables)], 0)
        b.input_ids = torch.tensor(ids, device=device)
        want = m.forward(b)
        got = graphs.decode(pos, tables, ids)
        top = want.topk(2, dim=-1)
        for i, tok in enumerate(got):   # (a width bucket splits keys otherwise: near ties may flip)
            assert tok == int(top.indices[i, 0]) or \
                want[i, tok] >= top.values[i, 0] - 10 * 2.0 ** -8 * want.abs().max()
