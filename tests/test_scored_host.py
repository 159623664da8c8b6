"""Attention with changed scores, shared prefixes and block norms without a GPU:
what the wrappers and the C entries refuse, which block_norms calls reach a launch,
the groups of a batch, and the oracle against torch's softmax."""
import ctypes
import math

import pytest
import torch

from nanopd_amd import _lib
from nanopd_amd import paged_kernels as pk
from oracle import scored_oracle as S
from .test_layer_ops_host import OnGpu, on_gpu


# -- the wrappers' refusals -------------------------------------------------------

class OnDevice(OnGpu):
    device = property(lambda self: torch.device("cuda", self.gpu))


def dev(*shape, dtype=torch.bfloat16, gpu=0):
    t = torch.ones(*shape, dtype=dtype).as_subclass(OnDevice)
    t.gpu = gpu
    return t


def i32(*shape):
    return dev(*shape, dtype=torch.int32)


def f32(*shape):
    return dev(*shape, dtype=torch.float32)


@pytest.fixture
def called(monkeypatch):
    calls = []
    monkeypatch.setattr(pk, "_call_on", lambda device, name, *args: calls.append((name, args)))
    return calls


def decode_args(**change):
    a = dict(out=dev(3, 8, 64), query=dev(3, 8, 64), key_cache=dev(9, 2, 16, 64),
             value_cache=dev(9, 2, 16, 64), block_tables=i32(3, 4), seq_lens=i32(3), scale=0.125,
             block_size=16, max_num_blocks_per_seq=4)
    a.update(change)
    return a


def shared_args(**change):
    return decode_args(**{"cu_groups": i32(3), "shared_lens": i32(2), "max_shared_len": 32, **change})


def prefill_args(**change):
    a = decode_args(out=dev(7, 8, 64), query=dev(7, 8, 64), cu_seqlens_q=i32(4),
                    context_lens=i32(3), max_q_len=5)
    del a["seq_lens"]
    a.update(change)
    return a


OPS = [(pk.paged_attention_scored, decode_args, "npd_paged_attention_scored"),
       (pk.paged_attention_shared, shared_args, "npd_paged_attention_shared"),
       (pk.paged_prefill_attention_scored, prefill_args, "npd_paged_prefill_scored")]


@pytest.mark.parametrize("op,args,name", OPS)
def test_calls_that_fit_reach_the_library(called, op, args, name):
    ws = dev(2 ** 24, dtype=torch.uint8)
    op(**args(workspace=ws))
    op(**args(workspace=ws, softcap=30.0, alibi_slopes=f32(8), window=5))
    assert [c[0] for c in called] == [name] * 2


WRONG = [
    dict(query=torch.ones(3, 8, 64)),                              # not on a GPU
    dict(query=dev(3, 512)),
    dict(query=dev(3, 8, 64, gpu=1)),
    dict(out=dev(4, 8, 64)),
    dict(out=dev(3, 8, 64, dtype=torch.float16)),
    dict(query=dev(3, 7, 64), out=dev(3, 7, 64)),            # 7 heads on 2
    dict(query=dev(3, 8, 32), out=dev(3, 8, 32)),
    dict(key_cache=dev(9, 2, 16, 64, dtype=torch.float16)),
    dict(value_cache=dev(8, 2, 16, 64)),
    dict(key_cache=dev(9, 2, 16, 64, gpu=1)),
    dict(block_size=8),
    dict(block_tables=i32(3, 5)),
    dict(block_tables=i32(2, 4)),
    dict(block_tables=i32(3, 4).long()),
    dict(alibi_slopes=dev(8)),
    dict(alibi_slopes=f32(4)),
    dict(alibi_slopes=torch.ones(8)),
    dict(k_scale=f32(2)),                                          # an FP8 pool wants both, and e4m3
    dict(k_scale=f32(2), v_scale=f32(2)),
    dict(workspace=dev(0, dtype=torch.uint8), block_tables=i32(3, 900),
         max_num_blocks_per_seq=900, max_context_len=14400, max_q_len=7),
]


@pytest.mark.parametrize("wrong", range(len(WRONG)))
@pytest.mark.parametrize("op,args,name", OPS)
def test_wrappers_refuse(called, op, args, name, wrong):
    change = dict(WRONG[wrong])
    if op is pk.paged_prefill_attention_scored:
        for k in ("query", "out"):   # seven rows of three sequences
            if k in change and change[k].dim() == 3 and change[k].size(0) == 3:
                t = change[k]
                change[k] = (dev(7, *t.shape[1:], dtype=t.dtype, gpu=t.gpu) if isinstance(t, OnDevice)
                             else torch.ones(7, *t.shape[1:]))
    else:
        change.pop("max_context_len", None)
        change.pop("max_q_len", None)
    with pytest.raises(RuntimeError):
        op(**args(**change))
    assert not called


@pytest.mark.parametrize("op,args,names", [
    (pk.paged_attention_scored, decode_args, {"seq_lens": 3, "first_keys": 3, "prefix_lens": 3}),
    (pk.paged_attention_shared, shared_args, {"seq_lens": 3, "cu_groups": None, "shared_lens": 2}),
    (pk.paged_prefill_attention_scored, prefill_args,
     {"cu_seqlens_q": None, "context_lens": 3, "first_keys": 7, "prefix_lens": 3}),
])
def test_wrappers_refuse_vectors(called, op, args, names):
    for name, n in names.items():
        bad = [i32(3, 3), f32(8), i32(16)[::2], torch.ones(8, dtype=torch.int32), "x"]
        if n is not None:
            bad.append(i32(n - 1))
        else:
            bad.append(i32(0))
        if name not in ("first_keys", "prefix_lens"):
            bad.append(None)
        for b in bad:
            with pytest.raises(RuntimeError):
                op(**args(**{name: b}))
    assert not called


@pytest.mark.parametrize("op,args,name", OPS)
def test_empty_calls_launch_nothing(called, op, args, name):
    e = dev(0, 8, 64)
    op(**args(query=e, out=e))
    assert not called


# -- the C entries ------------------------------------------------------------------

fake = 0x10000   # never dereferenced: validation fails first
no_gpu = pytest.mark.skipif(torch.cuda.is_available(),
                            reason="fake pointers: never run where a launch could happen")
F = ctypes.c_float


def c_decode(out=fake, q=fake, k=fake, v=fake, bt=fake, sl=fake, s=4, h=8, kv=2, d=64, nb=64, bs=16,
             mb=256, scale=0.1, cap=0.0, slopes=None, window=0, first=None, pre=None, ks=None, vs=None,
             strides=(512, 64, 512, 64), ws=None, wsb=0, dtype=1):
    return _lib.load().npd_paged_attention_scored(out, q, k, v, bt, sl, s, h, kv, d, nb, bs, mb, F(scale),
                                                  F(cap), slopes, window, first, pre, ks, vs, *strides, ws,
                                                  wsb, dtype, None)


def c_shared(out=fake, q=fake, k=fake, v=fake, bt=fake, sl=fake, cu=fake, sh=fake, s=4, g=2, msh=100, h=8,
             kv=2, d=64, nb=64, bs=16, mb=256, scale=0.1, cap=0.0, slopes=None, window=0, ks=None, vs=None,
             strides=(512, 64, 512, 64), ws=None, wsb=0, dtype=1):
    return _lib.load().npd_paged_attention_shared(out, q, k, v, bt, sl, cu, sh, s, g, msh, h, kv, d, nb, bs,
                                                  mb, F(scale), F(cap), slopes, window, ks, vs, *strides,
                                                  ws, wsb, dtype, None)


def c_prefill(out=fake, q=fake, k=fake, v=fake, bt=fake, cu=fake, sl=fake, s=4, tq=40, h=8, kv=2, d=64,
              nb=64, bs=16, mb=256, mq=20, mc=3000, scale=0.1, cap=0.0, slopes=None, window=0, first=None,
              pre=None, ks=None, vs=None, strides=(512, 64, 512, 64), ws=None, wsb=0, dtype=1):
    return _lib.load().npd_paged_prefill_scored(out, q, k, v, bt, cu, sl, s, tq, h, kv, d, nb, bs, mb, mq,
                                                mc, F(scale), F(cap), slopes, window, first, pre, ks, vs,
                                                *strides, ws, wsb, dtype, None)


INVALID, DTYPE, ALIGN, WORKSPACE = -1, -2, -3, -4
BAD = [
    (dict(dtype=7), DTYPE, b"dtype"), (dict(s=-1), INVALID, b"sizes"), (dict(h=0), INVALID, b"sizes"),
    (dict(h=9), INVALID, b"multiple"), (dict(d=60), INVALID, b"head_dim"), (dict(d=24), INVALID, b"head_dim"),
    (dict(d=264), INVALID, b"head_dim"), (dict(d=72, ks=fake, vs=fake), INVALID, b"head_dim"),
    (dict(nb=2 ** 30), INVALID, b"int32"), (dict(mb=2 ** 30), INVALID, b"int32"),
    (dict(s=2 ** 29), INVALID, b"rows"), (dict(scale=0.0), INVALID, b"scale"),
    (dict(scale=math.nan), INVALID, b"scale"), (dict(scale=math.inf), INVALID, b"scale"),
    (dict(cap=-1.0), INVALID, b"softcap"), (dict(cap=math.nan), INVALID, b"softcap"),
    (dict(cap=math.inf), INVALID, b"softcap"), (dict(cap=1e-38), INVALID, b"softcap"),
    (dict(window=-1), INVALID, b"window"), (dict(window=2 ** 31), INVALID, b"window"),
    (dict(strides=(516, 64, 512, 64)), ALIGN, b"strides"), (dict(strides=(512, 64, 512, -64)), ALIGN, b"strides"),
    (dict(out=None), INVALID, b"null"), (dict(bt=None), INVALID, b"null"), (dict(sl=None), INVALID, b"null"),
    (dict(ks=fake), INVALID, b"both"), (dict(vs=fake), INVALID, b"both"),
    (dict(q=fake + 8), ALIGN, b"aligned"), (dict(k=fake + 8), ALIGN, b"aligned"),
    (dict(), WORKSPACE, b"workspace"), (dict(ws=fake, wsb=100), WORKSPACE, b"workspace"),
    (dict(ws=fake + 16, wsb=2 ** 40), ALIGN, b"workspace"),
]


@no_gpu
@pytest.mark.parametrize("entry", [c_decode, c_shared, c_prefill])
@pytest.mark.parametrize("bad", range(len(BAD)))
def test_c_entries_refuse(entry, bad):
    change, rc, word = BAD[bad]
    assert entry(**change) == rc
    assert word in _lib.load().npd_last_error()


@no_gpu
def test_c_entries_refuse_their_own():
    err = _lib.load().npd_last_error
    for change in (dict(g=0), dict(g=2 ** 31), dict(msh=-1)):
        assert c_shared(**change) == INVALID and b"groups" in err()
    assert c_shared(cu=None) == INVALID and c_shared(sh=None) == INVALID and b"null" in err()
    # (as many groups as there can be: their costs are counted in coarser steps)
    assert c_shared(g=2 ** 31 - 1, msh=4096, s=3000, mb=2 ** 20) == WORKSPACE
    assert c_shared(msh=2 ** 62, s=3000) == WORKSPACE
    assert c_prefill(cu=None) == INVALID and b"null" in err()
    for change in (dict(mq=0), dict(mq=2 ** 31), dict(mc=-1)):
        assert c_prefill(**change) == INVALID and b"max_q_len" in err()
    assert c_prefill(s=2 ** 28, tq=2 ** 28, mq=2 ** 28 - 1, wsb=0) != 0


@no_gpu
def test_empty_batches_return_ok():
    assert c_decode(s=0, out=None) == 0
    assert c_shared(s=0, out=None) == 0
    assert c_prefill(s=0, out=None) == 0
    assert c_prefill(tq=0, out=None) == 0


@no_gpu
def test_block_norms_entry_refuses():
    lib = _lib.load()

    def call(out=fake, h=fake, x=fake, delta=fake, pw=fake, w=fake, gate=None, gr=0, gc=0, rows=4, width=64,
             rs=1.0, eps=1e-6, dtype=1):
        return lib.npd_block_norms(out, h, x, delta, pw, w, gate, gr, gc, rows, width, F(rs), F(eps), dtype,
                                   None)

    assert call(dtype=9) == DTYPE
    assert call(width=60) != 0 and call(width=8200) != 0 and call(rows=-1) != 0
    assert call(x=None) != 0 and call(delta=None) != 0 and call(out=None) != 0
    assert call(h=None) != 0 and call(x=fake + 2) != 0 and call(pw=fake + 8) != 0
    assert call(rows=0) == 0


def test_workspace_sizes():
    # nothing to merge: one part per unit
    assert pk.scored_workspace_bytes(4, 32, 8, 128, 16, 16) == 0
    a = pk.scored_workspace_bytes(4, 32, 8, 128, 16, 512)
    assert 0 < a < pk.scored_workspace_bytes(4, 32, 8, 128, 16, 4096)
    # a window bounds the parts, unless prefix keys stay visible behind it
    assert pk.scored_workspace_bytes(4, 32, 8, 128, 16, 512, window=128) == 0
    assert pk.scored_workspace_bytes(4, 32, 8, 128, 16, 512, window=128, prefix=True) == a
    assert pk.shared_workspace_bytes(4, 32, 8, 128, 16, 512, 1, 4096) > 0
    # shared keys are counted to the table's end
    assert pk.shared_workspace_bytes(64, 32, 8, 128, 16, 512, 1, 2 ** 62) == \
        pk.shared_workspace_bytes(64, 32, 8, 128, 16, 512, 1, 8192)
    assert pk.prefill_scored_workspace_bytes(1, 40000, 32, 8, 128, 40000, 40000) == 0   # whole tiles
    assert pk.prefill_scored_workspace_bytes(2, 600, 32, 8, 128, 300, 4000) > 0
    for bad in ((0, 8, 2, 64, 16, 4), (4, 8, 2, 64, 16, 2 ** 31), (2 ** 31, 8, 2, 64, 16, 4)):
        assert pk.scored_workspace_bytes(*bad) == 0


# -- block_norms -------------------------------------------------------------------

@pytest.fixture
def launches(monkeypatch):
    calls = []
    monkeypatch.setattr(pk, "_call_on", lambda device, name, *args: calls.append((name, args)))
    return calls


def test_block_norms_launches_what_fits(launches):
    x, d, w = on_gpu(3, 64), on_gpu(3, 64), on_gpu(64)
    pk.block_norms(x, d, w, w, 1e-6)
    assert pk.block_norms(x, d, None, None, 1e-6) is None
    for gate in (on_gpu(64), on_gpu(3, 1), on_gpu(3, 64), on_gpu(1, 64), on_gpu(1, 1)):
        pk.block_norms(x, d, w, w, 1e-6, gate=gate)
    pk.block_norms(x, d, w, w, 1e-6, x_out=d)
    assert [c[0] for c in launches] == ["npd_block_norms"] * 8


@pytest.mark.parametrize("change", [
    dict(delta=on_gpu(2, 64)), dict(post_weight=on_gpu(32)), dict(weight=on_gpu(128)),
    dict(x_out=on_gpu(4, 64)), dict(gate=on_gpu(32)), dict(gate=on_gpu(5, 64)),
])
def test_block_norms_refuses_what_does_not_fit(launches, change):
    a = dict(x=on_gpu(3, 64), delta=on_gpu(3, 64), post_weight=on_gpu(64), weight=on_gpu(64), eps=1e-6)
    a.update(change)
    with pytest.raises(RuntimeError):
        pk.block_norms(**a)
    assert not launches


def test_block_norms_launches_nothing_across_gpus(launches):
    x, w = on_gpu(3, 64), on_gpu(64)
    for kw in (dict(delta=on_gpu(3, 64, gpu=1)), dict(delta=on_gpu(3, 64), gate=on_gpu(64, gpu=1))):
        pk.block_norms(x, post_weight=w, weight=w, eps=1e-6, **kw)   # (refused for real tensors of two)
    assert not launches


def plain_norms(x, delta, pw, w, eps, gate, scale):
    def norm(t):
        return t * torch.rsqrt(t.pow(2).mean(-1, keepdim=True) + eps)
    d = norm(delta) * pw
    y = scale * x + gate * d
    return y, norm(y) * w


def test_block_norms_gradients(launches):
    """Calls that record a gradient run as torch operations: against the formula's
    own gradients and against differences."""
    g = torch.Generator().manual_seed(2)
    t = {n: torch.randn(*s, generator=g, dtype=torch.float64).requires_grad_()
         for n, s in dict(x=(3, 16), delta=(3, 16), pw=(16,), w=(16,), gate=(16,)).items()}

    def run(x, delta, pw, w, gate):
        y = torch.empty_like(x)
        h = pk.block_norms(x, delta, pw, w, 1e-3, gate=gate, residual_scale=0.5, x_out=y)
        return y.double(), h.double()

    co = [torch.randn(3, 16, generator=g, dtype=torch.float64) for _ in range(2)]
    got = torch.autograd.grad(run(*t.values()), list(t.values()), co)
    ref = torch.autograd.grad(plain_norms(*[t[n] for n in ("x", "delta", "pw", "w")], 1e-3, t["gate"], 0.5),
                              list(t.values()), co)
    # (fp32 inside: each of about 100 operations on values below 30 rounds by 2^-24)
    for a, b in zip(got, ref):
        assert (a - b).abs().max() <= 100 * 30 * 2.0 ** -24
    for i, name in enumerate(t):   # central differences of the 64-bit formula: error h^2 times thirds
        v = torch.randn(t[name].shape, generator=g, dtype=torch.float64)
        ends = []
        for s in (1e-4, -1e-4):
            u = {n: a.detach() + (s * v if n == name else 0) for n, a in t.items()}
            y = plain_norms(u["x"], u["delta"], u["pw"], u["w"], 1e-3, u["gate"], 0.5)
            ends.append(sum((a * b).sum() for a, b in zip(y, co)))
        assert abs((ends[0] - ends[1]) / 2e-4 - (got[i] * v).sum()) <= 1e-3
    assert not launches


# -- groups of a batch ----------------------------------------------------------------

def test_find_shared_prefixes():
    def find(tables, lens):
        p = pk.find_shared_prefixes(tables, lens, 16, "cpu")
        return None if p is None else (p.cu_groups.tolist(), p.shared_lens.tolist(), p.max_shared_len)

    assert find([], []) is None
    assert find([[1, 2]], [32]) is None
    assert find([[1, 2], [3, 4]], [32, 32]) is None
    assert find([[1, 2, 3], [1, 2, 4]], [40, 41]) == ([0, 2], [32], 32)
    # a shared block that is not full of one's tokens is not shared
    assert find([[1, 2, 3], [1, 2, 4]], [40, 31]) == ([0, 2], [16], 16)
    assert find([[1, 2], [1, 2]], [15, 15]) is None
    # the group ends where a sequence would halve it, and only neighbours share
    long = list(range(10))
    assert find([long, long, [0, 1, 99], long], [160, 160, 48, 160]) == \
        ([0, 2, 4], [160, 32], 160)
    assert find([[7], [1, 2, 3], [1, 2, 5], [9, 9]], [16, 48, 48, 20]) == ([0, 1, 3, 4], [0, 32, 0], 32)


# -- the oracle --------------------------------------------------------------------------

def test_oracle_is_a_softmax():
    g = torch.Generator().manual_seed(0)
    q = torch.randn(5, 4, 32, generator=g, dtype=torch.float64)
    k, v = (torch.randn(9, 2, 32, generator=g, dtype=torch.float64) for _ in range(2))
    pos = torch.arange(4, 9)
    out, _ = S.attend(q, k, v, pos, 9, 0.3, softcap=2.0, slopes=torch.full((4,), 0.1), window=3, prefix=1)
    for t in range(5):
        for h in range(4):
            s = [2.0 * math.tanh(0.3 * float(q[t, h] @ k[j, h // 2]) / 2.0) - 0.1 * abs(int(pos[t]) - j)
                 for j in range(9)]
            seen = [j for j in range(9) if j <= pos[t] and pos[t] - j < 3 or j < 1]
            p = torch.softmax(torch.tensor([s[j] for j in seen], dtype=torch.float64), 0)
            want = sum(p[i] * v[j, h // 2] for i, j in enumerate(seen))
            assert (out[t, h] - want).abs().max() < 1e-6    # (slopes are fp32)
    empty, _ = S.attend(q, k, v, pos, 9, 0.3, first=torch.full((5,), 9))
    assert (empty == 0).all()
