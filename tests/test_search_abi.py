"""The search entry points without a GPU: workspace sizes, refusals (all before any device call), the
binding's checks, and the oracle's own properties."""
import numpy as np
import pytest

import densecore_amd as dc
from oracle import search as S

OK, INVALID, UNSUPPORTED, BAD_SHAPE, MISALIGNED, WORKSPACE, NO_DEVICE = 0, -1, -2, -3, -4, -5, -7
F32, F16, Q8_0 = 0, 1, 8
BIG = 0x10000000


def no_gpu():
    import torch
    return not torch.cuda.is_available()


def tree(ct=F16, k=0x1000, v=0x2000, blocks=8, layers=2, layer=1, tables=0x3000, stride=4, width=4, past=0x4000,
         max_past=40, drafts=0x5000, mask=0x6000, heads=8, kv=2, hd=64, q=0x100000, qs=None, kc=0x200000, vc=0x300000,
         kvs=None, seqs=2, tokens=3, scale=0.125, out=0x400000, outs=None, ws=BIG, wsb=1 << 30):
    qs = heads * hd * 4 if qs is None else qs
    kvs = kv * hd * 4 if kvs is None else kvs
    outs = heads * hd * 4 if outs is None else outs
    return dc.lib().dcq_kv_tree_attention(ct, k, v, blocks, layers, layer, tables, stride, width, past, max_past, drafts,
                                          mask, heads, kv, hd, q, qs, kc, vc, kvs, seqs, tokens, scale, out, outs, ws,
                                          wsb, None)


@pytest.mark.parametrize("kw,want", [
    (dict(ct=2), UNSUPPORTED), (dict(hd=96), UNSUPPORTED), (dict(heads=7), BAD_SHAPE), (dict(heads=0), BAD_SHAPE),
    (dict(tokens=0), BAD_SHAPE), (dict(tokens=1025), BAD_SHAPE), (dict(seqs=0), BAD_SHAPE), (dict(seqs=65536), BAD_SHAPE),
    (dict(max_past=-1), BAD_SHAPE), (dict(max_past=(1 << 24) + 1), BAD_SHAPE), (dict(layer=2), BAD_SHAPE),
    (dict(blocks=0), BAD_SHAPE), (dict(k=None), INVALID), (dict(v=None), INVALID), (dict(tables=None), INVALID),
    (dict(width=-1), BAD_SHAPE), (dict(stride=3), INVALID), (dict(past=None), INVALID), (dict(q=None), INVALID),
    (dict(kc=None), INVALID), (dict(vc=None), INVALID), (dict(out=None), INVALID), (dict(scale=float("nan")), INVALID),
    (dict(scale=float("inf")), INVALID), (dict(qs=16), INVALID), (dict(kvs=16), INVALID), (dict(outs=16), INVALID),
    (dict(q=0x100004), MISALIGNED), (dict(kc=0x200008), MISALIGNED), (dict(qs=2052), MISALIGNED),
    (dict(past=0x4002), MISALIGNED), (dict(mask=0x6004), MISALIGNED), (dict(drafts=0x5001), MISALIGNED),
    (dict(out=0x100100), INVALID), (dict(out=0x200000), INVALID),
    (dict(max_past=100000, ws=None), WORKSPACE), (dict(max_past=100000, wsb=256), WORKSPACE),
    (dict(max_past=100000, ws=BIG + 16), MISALIGNED),
])
def test_tree_attention_refusals(kw, want):
    assert tree(**kw) == want


def test_tree_attention_workspace():
    size = dc.kv_tree_attention_workspace_size
    assert size(8, 2, 64, 1, 1, 0) == 0 and size(8, 2, 64, 1, 4, 100) == 0
    assert size(8, 2, 64, 1, 4, 100000) > 0
    assert size(7, 2, 64, 1, 4, 100) == 0 and size(8, 2, 80, 1, 4, 100) == 0
    if no_gpu():
        assert tree() == NO_DEVICE
        assert tree(tables=None, width=0, drafts=None, mask=None, max_past=0) == NO_DEVICE


def path(ct=F32, k=0x1000, v=0x2000, blocks=8, layers=2, elems=64, tables=0x3000, stride=4, width=4, past=0x4000,
         pth=0x5000, ps=3, n=3, n_path=0x6000, kc=0x100000, vc=0x200000, ls=4096, rs=256, seqs=2, tokens=3):
    return dc.lib().dcq_kv_write_path(ct, k, v, blocks, layers, elems, tables, stride, width, past, pth, ps, n, n_path,
                                      kc, vc, ls, rs, seqs, tokens, None)


@pytest.mark.parametrize("kw,want", [
    (dict(ct=3), UNSUPPORTED), (dict(elems=40), BAD_SHAPE), (dict(layers=0), BAD_SHAPE), (dict(layers=65536), BAD_SHAPE),
    (dict(seqs=0), BAD_SHAPE), (dict(tokens=0), BAD_SHAPE), (dict(n=-1), BAD_SHAPE), (dict(n=0), OK),
    (dict(k=None), INVALID), (dict(v=None), INVALID), (dict(past=None), INVALID), (dict(pth=None), INVALID),
    (dict(kc=None), INVALID), (dict(vc=None), INVALID), (dict(ps=2), INVALID), (dict(stride=2), INVALID),
    (dict(rs=128), INVALID), (dict(ls=1024), INVALID), (dict(rs=264, ls=8192), MISALIGNED), (dict(ls=4104), MISALIGNED),
    (dict(kc=0x100004), MISALIGNED), (dict(pth=0x5002), MISALIGNED), (dict(tables=0x3001), MISALIGNED),
])
def test_write_path_refusals(kw, want):
    assert path(**kw) == want


def fork(ct=F16, k=0x1000, v=0x2000, blocks=8, layers=2, elems=64, tables=0x3000, stride=4, width=4, lengths=0x4000,
         seqs=2, parents=0x5000, children=3, refs=0x6000, to=0x7000, tos=4, lo=0x8000, ro=0x9000, missing=0xa000,
         ws=BIG, wsb=1 << 20):
    return dc.lib().dcq_kv_fork(ct, k, v, blocks, layers, elems, tables, stride, width, lengths, seqs, parents, children,
                                refs, to, tos, lo, ro, missing, ws, wsb, None)


@pytest.mark.parametrize("kw,want", [
    (dict(ct=9), UNSUPPORTED), (dict(blocks=0), BAD_SHAPE), (dict(width=0), BAD_SHAPE), (dict(seqs=0), BAD_SHAPE),
    (dict(children=0), BAD_SHAPE), (dict(children=4097), BAD_SHAPE), (dict(elems=33), BAD_SHAPE),
    (dict(lengths=None), INVALID), (dict(parents=None), INVALID), (dict(refs=None), INVALID), (dict(to=None), INVALID),
    (dict(lo=None), INVALID), (dict(ro=None), INVALID), (dict(missing=None), INVALID), (dict(stride=3), INVALID),
    (dict(tos=3), INVALID), (dict(to=0x3000), INVALID), (dict(ro=0x6000), INVALID), (dict(lo=0x4004), INVALID),
    (dict(missing=0x5008), INVALID), (dict(ro=0x9002), MISALIGNED), (dict(lengths=0x4001), MISALIGNED),
    (dict(ws=None), WORKSPACE), (dict(wsb=16), WORKSPACE), (dict(ws=BIG + 4), MISALIGNED), (dict(v=0x2008), MISALIGNED),
])
def test_fork_refusals(kw, want):
    assert fork(**kw) == want


def compact(ct=F16, k=0x1000, v=0x2000, blocks=8, layers=2, elems=64, tables=0x3000, stride=4, width=4, lengths=0x4000,
            seqs=2, refs=0x6000, to=0x7000, tos=4, ro=0x9000, live=0xa000, ws=BIG, wsb=1 << 20):
    return dc.lib().dcq_kv_compact(ct, k, v, blocks, layers, elems, tables, stride, width, lengths, seqs, refs, to, tos,
                                   ro, live, ws, wsb, None)


@pytest.mark.parametrize("kw,want", [
    (dict(ct=9), UNSUPPORTED), (dict(blocks=-1), BAD_SHAPE), (dict(width=0), BAD_SHAPE), (dict(seqs=0), BAD_SHAPE),
    (dict(lengths=None), INVALID), (dict(refs=None), INVALID), (dict(to=None), INVALID), (dict(ro=None), INVALID),
    (dict(live=None), INVALID), (dict(tos=3), INVALID), (dict(to=0x3010), INVALID), (dict(ro=0x6004), INVALID),
    (dict(live=0xa001), MISALIGNED), (dict(ws=None), WORKSPACE), (dict(wsb=16), WORKSPACE),
])
def test_compact_refusals(kw, want):
    assert compact(**kw) == want


def beam(t=F32, x=0x1000, xs=400, b=2, w=3, v=100, bs=0x100000, n=4, sc=0x200000, pa=0x300000, to=0x400000, ws=BIG,
         wsb=1 << 20):
    return dc.lib().dcq_beam_select(t, x, xs, b, w, v, bs, n, sc, pa, to, ws, wsb, None)


@pytest.mark.parametrize("kw,want", [
    (dict(t=8), UNSUPPORTED), (dict(b=0), BAD_SHAPE), (dict(w=0), BAD_SHAPE), (dict(w=257), BAD_SHAPE),
    (dict(b=30000), BAD_SHAPE), (dict(v=0), BAD_SHAPE), (dict(v=(1 << 24) + 1), BAD_SHAPE), (dict(n=0), BAD_SHAPE),
    (dict(n=65), BAD_SHAPE), (dict(x=None), INVALID), (dict(bs=None), INVALID), (dict(sc=None), INVALID),
    (dict(pa=None), INVALID), (dict(to=None), INVALID), (dict(xs=396), INVALID), (dict(xs=402), MISALIGNED),
    (dict(x=0x1002), MISALIGNED), (dict(t=F16, x=0x1001), MISALIGNED), (dict(sc=0x1000), INVALID),
    (dict(to=0x100004), INVALID), (dict(ws=None), WORKSPACE), (dict(wsb=64), WORKSPACE), (dict(ws=BIG + 128), MISALIGNED),
])
def test_beam_select_refusals(kw, want):
    assert beam(**kw) == want


W = dict(max_past=100000, ws=None)  # a call that goes as far as the workspace's check


@pytest.mark.parametrize("kw,want", [
    (dict(q=0x100000, qs=8192, out=0x100800, outs=8192, **W), WORKSPACE),   # outputs beside the queries in wider rows
    (dict(q=0x100800, qs=8192, out=0x100000, outs=8192, **W), WORKSPACE),
    (dict(q=0x100000, qs=8192, out=0x101800, outs=8192, **W), WORKSPACE),
    (dict(q=0x100000, qs=8192, out=0x100000 + 6 * 8192, outs=8192, **W), WORKSPACE),
    (dict(q=0x100000, qs=8192, out=0x1007fc, outs=8192, **W), INVALID),     # a row's last element
    (dict(q=0x100000, qs=8192, out=0x101804, outs=8192, **W), INVALID),     # the next row's first one
    (dict(q=0x101000, qs=8192, out=0x1007fc, outs=8192, **W), WORKSPACE),
    (dict(q=0x101000, qs=8192, out=0x100804, outs=8192, **W), INVALID),
    (dict(q=0x100000, qs=8192, out=0x100800, outs=4096, **W), INVALID),     # other strides
])
def test_tree_attention_overlaps(kw, want):
    assert tree(**kw) == want


@pytest.mark.parametrize("kw,want", [
    (dict(stride=8, to=0x3010, tos=8, ws=None), WORKSPACE),   # two tables in turn, in wider rows
    (dict(stride=8, to=0x300c, tos=8, ws=None), INVALID), (dict(stride=8, to=0x3014, tos=8, ws=None), INVALID),
])
def test_fork_and_compact_tables_in_wider_rows(kw, want):
    assert fork(**kw) == want and compact(**kw) == want


@pytest.mark.parametrize("kw,want", [
    (dict(out=0x3000, **W), INVALID), (dict(out=0x4004, **W), INVALID), (dict(out=0x6000, **W), INVALID),
    (dict(max_past=100000, ws=0x400000), INVALID), (dict(max_past=100000, ws=0x100000), INVALID),
    (dict(max_past=100000, ws=0x4000, wsb=1 << 26), INVALID),
])
def test_tree_attention_output_and_workspace_overlaps(kw, want):
    assert tree(**kw) == want


@pytest.mark.parametrize("kw,want", [
    (dict(lo=0x7000), INVALID), (dict(ro=0x8008), INVALID), (dict(missing=0x901c), INVALID), (dict(missing=0x7000), INVALID),
    (dict(ws=0x7000), INVALID), (dict(ws=0x2f00), INVALID), (dict(ws=0x6000), INVALID), (dict(ws=0x8f00), INVALID),
])
def test_fork_overlaps(kw, want):
    assert fork(**kw) == want


@pytest.mark.parametrize("kw,want", [
    (dict(ro=0x7010), INVALID), (dict(live=0x9004), INVALID), (dict(live=0x7000), INVALID),
    (dict(ws=0x7000), INVALID), (dict(ws=0x4000), INVALID), (dict(ws=0x8f00), INVALID),
])
def test_compact_overlaps(kw, want):
    assert compact(**kw) == want


@pytest.mark.parametrize("kw,want", [
    (dict(pa=0x20001c), INVALID), (dict(to=0x300000), INVALID), (dict(to=0x200000), INVALID), (dict(ws=0x200000), INVALID),
    (dict(ws=0x1000), INVALID), (dict(ws=0x100000), INVALID), (dict(pa=0x200020, ws=None), WORKSPACE),
])
def test_beam_select_overlaps(kw, want):
    assert beam(**kw) == want


GRIDS = [
    # one workgroup of 256 threads per (sequence, KV head): 2^24 workgroups are 2^32 threads, one more than a launch has
    (dict(seqs=65535, tokens=1, heads=257, kv=257), BAD_SHAPE), (dict(seqs=65535, tokens=1, heads=256, kv=256), None),
    (dict(seqs=4096, tokens=1, heads=4096, kv=4096), BAD_SHAPE),
    (dict(seqs=4096, tokens=1, heads=4096, kv=4096, max_past=100000, ct=F32), BAD_SHAPE),
    (dict(seqs=65535, tokens=2, heads=512, kv=128), None), (dict(seqs=65535, tokens=9, heads=192, kv=48), None),
    # blocks of rows: the workgroups of the drafted keys come on top
    (dict(seqs=65535, tokens=17, heads=120, kv=120, max_past=1000, hd=128), BAD_SHAPE),
    (dict(seqs=20000, tokens=17, heads=120, kv=120, max_past=1000, hd=128), None),
    # the merge: a thread for four elements
    (dict(seqs=16384, tokens=1024, heads=4, kv=1, hd=256, max_past=0), BAD_SHAPE),
    (dict(seqs=16383, tokens=1024, heads=4, kv=1, hd=256, max_past=0), None),
    (dict(seqs=16384, tokens=1024, heads=8, kv=1, hd=128, max_past=0), BAD_SHAPE),
    (dict(seqs=16384, tokens=1024, heads=8, kv=1, hd=64, max_past=0), None),
    (dict(seqs=16385, tokens=1024, heads=8, kv=1, hd=64, max_past=0), BAD_SHAPE),
]


@pytest.mark.parametrize("kw,want", GRIDS)
def test_tree_attention_shapes_past_a_launch(kw, want):
    """What no launch holds is refused as a shape, what one just holds goes on to the next check (addresses of 0)."""
    assert tree(out=None, **kw) == (INVALID if want is None else want)


@pytest.mark.parametrize("seqs,n,want", [(65535, 257, BAD_SHAPE), (16384, 1024, BAD_SHAPE), (65535, 256, None), (16383, 1024, None)])
def test_write_path_shapes_past_a_launch(seqs, n, want):
    assert path(seqs=seqs, n=n, ps=n, past=None) == (INVALID if want is None else want)


def test_pages_past_a_launch():
    """Copies in more pieces than a launch counts (arenas of many terabytes)."""
    assert fork(blocks=8, layers=60000, elems=1 << 20, children=4096, ws=None) == BAD_SHAPE
    assert fork(layers=36, elems=1024, children=4096, to=0x100000, lo=0x200000, parents=0x300000, ws=None) == WORKSPACE
    assert compact(blocks=1 << 24, layers=36, elems=1 << 16, ws=None) == BAD_SHAPE
    assert compact(blocks=1 << 24, layers=36, elems=1024, ws=None, refs=0x80000000, ro=0x90000000) == WORKSPACE


def test_well_formed_calls_without_gpu_fail_loudly():
    if not no_gpu():
        pytest.skip("a GPU is present")
    assert path() == NO_DEVICE and path(n_path=None) == NO_DEVICE
    assert fork() == NO_DEVICE and compact() == NO_DEVICE
    assert beam() == NO_DEVICE and beam(t=F16, x=0x1002, xs=202) == NO_DEVICE


def test_binding_refuses_host_tensors_and_wrong_dtypes():
    import torch
    with pytest.raises(ValueError, match="GPU tensor"):
        dc.beam_select(torch.zeros(2, 8), torch.zeros(1, 2), 2)
    with pytest.raises(ValueError, match="dtype"):
        dc.beam_select(torch.zeros(2, 8, dtype=torch.float64), torch.zeros(1, 2), 2)
    cache = dc.PagedKVCache(F16, 4, 1, 2, 64, device="cpu")
    with pytest.raises(ValueError, match="GPU tensor"):
        cache.fork(torch.zeros(1, 2, dtype=torch.int32), torch.zeros(1, dtype=torch.int32),
                   torch.zeros(1, dtype=torch.int32), torch.zeros(4, dtype=torch.int32))
    with pytest.raises(ValueError, match="dtype"):
        cache.compact(torch.zeros(1, 2, dtype=torch.int64), torch.zeros(1, dtype=torch.int32),
                      torch.zeros(4, dtype=torch.int32))


def test_binding_names_arguments_that_are_no_tensors():
    from densecore_amd import _lib
    _lib._t()
    for value in ([3, 4], 7, None):
        with pytest.raises(ValueError, match="past: expected a torch tensor"):
            if not _lib._plain(value, _lib._I32, (2,)):
                _lib._checked("past", value, _lib._I32, (2,))
        with pytest.raises(ValueError, match="tables_out: expected a torch tensor" if value is not None else "tables"):
            _lib._rows_of("tables_out" if value is not None else "tables", value, _lib._I32, (2, 2))


def test_binding_refuses_memory_that_is_not_packed_on_the_gpu():
    """A workspace or an arena in host memory, or one that has fewer bytes than elements."""
    import torch
    from densecore_amd import _lib
    assert _lib._scratch(None) == (None, 0)
    for ws in (torch.empty(4096, dtype=torch.uint8), 4096, [0] * 4096):
        with pytest.raises(ValueError, match="contiguous GPU tensor"):
            _lib._scratch(ws)

    class Fake:  # what a GPU tensor answers, without a GPU
        is_cuda = True

        def __init__(self, t):
            self.t = t

        def __getattr__(self, name):
            return getattr(self.t, name)
    with pytest.raises(ValueError, match="contiguous GPU tensor"):
        _lib._scratch(Fake(torch.empty(1, dtype=torch.uint8).expand(1 << 20)))
    assert _lib._scratch(Fake(torch.empty(100, dtype=torch.int32)))[1] == 400
    cache = dc.PagedKVCache(F16, 4, 1, 2, 64, device="cpu")
    with pytest.raises(ValueError, match="contiguous GPU tensor"):
        cache._arenas()
    cache.k, cache.v = Fake(cache.k), Fake(cache.v[:100])
    with pytest.raises(ValueError, match="4 blocks need"):
        cache._arenas()


# ---------------------------------------------------------------- the oracle
def test_oracle_tree_of_a_chain_is_causal_attention(O):
    from oracle import kv as KV
    rng = np.random.default_rng(1)
    n, past, h, g, d = 5, 9, 4, 2, 64
    q, k, v = rng.normal(size=(n, h, d)), rng.normal(size=(past + n, g, d)), rng.normal(size=(past + n, g, d))
    want, (a, b) = KV.attention(q, k, v, past, 0.125)
    got, ga, gb = S.tree_attention(q, k[:past], v[:past], k[past:], v[past:], np.tril(np.ones((n, n), bool)), 0.125)
    assert np.allclose(got, want, rtol=1e-12) and np.allclose(ga, a) and np.allclose(gb, b)


def test_oracle_tree_reads_siblings_apart():
    rng = np.random.default_rng(2)
    q, k, v = rng.normal(size=(3, 2, 64)), rng.normal(size=(3, 2, 64)), rng.normal(size=(3, 2, 64))
    seen = np.array([[1, 0, 0], [1, 1, 0], [1, 0, 1]], bool)
    none = np.zeros((0, 2, 64))
    base = S.tree_attention(q, none, none, k, v, seen, 1.0)[0]
    k2, v2 = k.copy(), v.copy()
    k2[1], v2[1] = 1e9, np.nan  # token 1 is not an ancestor of token 2
    other = S.tree_attention(q, none, none, k2, v2, seen, 1.0)[0]
    assert np.array_equal(base[[0, 2]], other[[0, 2]]) and not np.array_equal(base[1], other[1])
    assert np.array_equal(base[0], v[[0]].repeat(1, 0)[0])
    assert not S.tree_attention(q, none, none, k, v, np.zeros((3, 3), bool), 1.0)[0].any()


def test_oracle_fork_shares_copies_and_frees():
    # one partial page (5) held by both parents' sequences only through sequence 0; sequence 1 ends on a full page
    tables, lengths, refs = [[3, 5], [4, 6]], [20, 32], [0, 0, 0, 1, 1, 1, 1, 0]
    t, n, r, missing, pairs = S.fork(tables, lengths, [0, 0, 1], refs)
    assert t == [[3, 5], [3, 0], [4, 6]] and n == [20, 20, 32] and missing == 0 and pairs == [(5, 0)]
    assert r == [1, 0, 0, 2, 1, 1, 1, 0]
    t, n, r, missing, pairs = S.fork(tables, lengths, [1, 7], refs)  # sequence 0 ends, parent 7 is none
    assert t == [[4, 6], [-1, -1]] and n == [32, 0] and r == [0, 0, 0, 0, 1, 0, 1, 0] and not pairs
    assert S.fork([[3, 5]], [20], [0, 0, 0], [1, 1, 1, 1, 1, 1])[3] == 2  # no free page
    # a holder beyond the call: even a single child copies
    assert S.fork([[3, 5]], [20], [0], [0, 0, 0, 1, 0, 2])[4] == [(5, 0)]


def test_oracle_compact_and_beams():
    t, r, live, pairs = S.compact([[6, 0], [4, 7]], [32, 20], [1, 0, 0, 0, 1, 0, 1, 2])
    assert live == 4 and pairs == [(4, 1), (6, 2), (7, 3)] and t == [[2, 0], [1, 3]] and r == [1, 1, 1, 2, 0, 0, 0, 0]
    x = np.zeros((2, 4))
    s, p, k = S.beam_select(x, np.array([[0.0, 0.0]]), 6)  # all equal: the lowest beam, then the lowest token
    assert p.tolist() == [[0, 0, 0, 0, 1, 1]] and k.tolist() == [[0, 1, 2, 3, 0, 1]] and np.allclose(s, -np.log(4))
