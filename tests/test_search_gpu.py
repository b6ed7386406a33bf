"""Search over the paged cache on the GPU, through the public binding, against oracle/search.py: whole numbers
and page bytes exactly, attention and scores within bounds counted from their roundings."""
import numpy as np
import pytest

import densecore_amd as dc
from oracle import search as S

pytestmark = pytest.mark.gpu

F32, F16, Q8_0 = 0, 1, 8
CACHE_TYPES = [F32, F16, Q8_0]


@pytest.fixture(scope="module")
def KV(O):
    from oracle import kv
    return kv


def to_dev(a, dev):
    import torch
    return torch.from_numpy(np.ascontiguousarray(a)).to(dev)


def i32(a, dev):
    return to_dev(np.asarray(a, np.int32), dev)


def to_host(t):
    import torch
    torch.cuda.synchronize()
    return t.cpu().numpy()


# ---------------------------------------------------------------- attention of drafted trees
def random_tree(n, rng, roots=0.2):
    seen = np.zeros((n, n), bool)
    for j in range(n):
        p = int(rng.integers(-1, j)) if j and rng.random() > roots else -1
        if p >= 0:
            seen[j] = seen[p]
        seen[j, j] = True
    return seen


class Tree:
    """Inputs of one call: histories of several sequences on shuffled pages, stale bytes in every unused slot."""

    def __init__(self, KV, ct, n, pasts, heads, kv, hd, seed, drafts=None, holes=(), n_layer=2, spread=1.0):
        rng = self.rng = np.random.default_rng(seed)
        self.ct, self.n, self.pasts, self.heads, self.kv, self.hd = ct, n, pasts, heads, kv, hd
        self.s, self.n_layer, self.layer, self.scale = len(pasts), n_layer, n_layer - 1, float(np.float32(hd ** -0.5))
        self.drafts = [n] * self.s if drafts is None else drafts
        row = kv * hd
        used = [(p + 15) // 16 for p in pasts]
        self.n_blocks = sum(used) + 2
        sb = KV.slot_bytes(ct, row)
        stale = {F32: np.float32(np.nan), F16: np.float16(np.inf), Q8_0: np.uint8(0xFF)}[ct]  # Q8_0: a NaN scale
        size = self.n_blocks * n_layer * 16 * sb
        self.arena = [np.full(size // stale.itemsize, stale).view(np.uint8).copy() for _ in range(2)]
        order, self.tables, at = rng.permutation(self.n_blocks), np.full((self.s, max(used + [1])), -1, np.int32), 0
        self.hist = []
        for b, p in enumerate(pasts):
            self.tables[b, :used[b]] = order[at:at + used[b]]
            at += used[b]
            rows = [(rng.normal(size=(p, row)) * spread).astype(np.float32) for _ in range(2)]
            for arena, x in zip(self.arena, rows):
                KV.write(ct, arena, n_layer, self.layer, self.tables[b], 0, x)
        for b, i in holes:
            self.tables[b, i] = -1
        empty = np.zeros((0, row), np.float32)
        for b, p in enumerate(pasts):
            self.hist.append([KV.gather(ct, arena, n_layer, self.layer, self.tables[b], p, empty).reshape(p, kv, hd)
                              for arena in self.arena])
        self.q = (rng.normal(size=(self.s, n, heads, hd)) * 2).astype(np.float32)
        self.kc, self.vc = (rng.normal(size=(self.s, n, kv, hd)).astype(np.float32) for _ in range(2))
        self.seen = np.stack([random_tree(n, rng) for _ in range(self.s)])

    def cache(self, dev):
        c = dc.PagedKVCache(self.ct, self.n_blocks, self.n_layer, self.kv, self.hd, device=dev)
        c.k.copy_(to_dev(self.arena[0], dev))
        c.v.copy_(to_dev(self.arena[1], dev))
        return c

    def args(self, dev):
        rows = self.s * self.n
        return (self.layer, to_dev(self.tables, dev), i32(self.pasts, dev), max(self.pasts),
                to_dev(self.q.reshape(rows, -1), dev), to_dev(self.kc.reshape(rows, -1), dev),
                to_dev(self.vc.reshape(rows, -1), dev), self.scale)

    def kwargs(self, dev):
        return {"mask": to_dev(np.stack([S.mask_words(m) for m in self.seen]), dev), "n_draft": i32(self.drafts, dev)}

    def run(self, dev):
        out = self.cache(dev).tree_attention(*self.args(dev), **self.kwargs(dev))
        return to_host(out).reshape(self.s, self.n, self.heads, self.hd)

    def run_and_check(self, dev):
        self.check(self.run(dev))

    def check(self, out):
        """Every row of every head: |out - ref| <= (2e-6 + 2^-21 B) |A| in the 2-norm. A score of magnitude up to B
        is off by the dropped parts of its operands' pieces (2^-22 of B for both), its sums' roundings (about as
        much) and the rounding of the scaled product, and moves its weight by as much; the weights' pieces (2^-22),
        exponentials and sums add a few of 2^-23 of A = sum_t p_t |v_t|, the sums over keys their roundings."""
        for b in range(self.s):
            m = self.drafts[b]
            ref, a, big = S.tree_attention(self.q[b, :m], *self.hist[b], self.kc[b, :m], self.vc[b, :m],
                                           self.seen[b, :m, :m], self.scale)
            assert not out[b, m:].any(), "rows past n_draft"
            nan = np.isnan(ref)
            assert np.array_equal(np.isnan(out[b, :m]), nan), f"sequence {b}: NaN in other places"
            with np.errstate(invalid="ignore"):
                err = np.linalg.norm(np.where(nan, 0, out[b, :m] - ref), axis=2)
            bound = (2e-6 + 2.0 ** -21 * big) * np.linalg.norm(np.where(nan, 0, a), axis=2)
            bad = ~(err <= bound) & ~nan.any(axis=2)
            assert not bad.any(), (f"sequence {b}: {int(bad.sum())} of {err.size} rows, first {np.argwhere(bad)[0]}, "
                                   f"worst {np.nanmax(err / np.maximum(bound, 1e-300)):.3g}")


TREES = [
    # (tokens, cached positions, heads, KV heads, head_dim)
    (1, [0], 1, 1, 64),                       # nothing cached: its own row alone
    (1, [1], 4, 4, 128),
    (1, [15, 16, 17, 31, 32, 33, 0], 8, 1, 256),   # the next token of several beams, one KV head
    (2, [127, 128, 129], 6, 2, 64),
    (7, [100], 16, 8, 128),                   # one user's small tree
    (5, [0, 3], 7, 1, 64),                    # 35 rows, a group of 7
    (24, [700, 5, 333], 32, 8, 128),          # 96 rows of a KV head
    (17, [513], 3, 3, 256),                   # a last tile of one row
    (64, [40], 4, 1, 64),                     # a whole mask word
    (65, [20, 1000], 4, 2, 128),              # two words, a second of one bit
    (100, [260], 8, 1, 64),                   # 800 rows
    (33, [2500], 8, 8, 64),                   # long, no group
    (3, [6000, 10], 8, 2, 128),               # many key splits, and a sequence with one
    (40, [1029], 16, 4, 256),
    (64, [1500, 300], 8, 2, 128),             # 256 rows
    (100, [257, 4100, 0], 3, 1, 128),         # 300 rows
    (9, [3001], 32, 8, 128),                  # 36 rows: a wave of four
]


@pytest.mark.parametrize("ct", CACHE_TYPES)
@pytest.mark.parametrize("n,pasts,heads,kv,hd", TREES)
def test_tree_attention(KV, dev, ct, n, pasts, heads, kv, hd):
    t = Tree(KV, ct, n, pasts, heads, kv, hd, seed=n + sum(pasts) + hd)
    print(f"tree ct={ct} n={n} pasts={pasts} heads={heads}/{kv} hd={hd}", flush=True)
    t.check(t.run(dev))


@pytest.mark.parametrize("ct", [F16, Q8_0])
@pytest.mark.parametrize("n,pasts,heads,kv,hd", [
    (17, [8200, 1, 515] + [0] * 29, 16, 1, 128),  # 272 rows: a second tile of 16, shares by the lengths
    (36, [0, 3, 9001] + [20] * 63, 4, 1, 64),     # 144 rows, more sequences than share
])
def test_tree_attention_long_shares(KV, dev, ct, n, pasts, heads, kv, hd):
    """More than 128 rows over shares of 1024 keys and more."""
    t = Tree(KV, ct, n, pasts, heads, kv, hd, seed=n + hd, n_layer=1)
    t.check(t.run(dev))


@pytest.mark.parametrize("ct", CACHE_TYPES)
@pytest.mark.parametrize("n,pasts,heads,kv,hd", [(11, [2001] * 9, 16, 4, 256), (12, [4000, 1200, 2800, 17], 32, 8, 256)])
def test_tree_attention_wide_heads_in_blocks(KV, dev, ct, n, pasts, heads, kv, hd):
    t = Tree(KV, ct, n, pasts, heads, kv, hd, seed=n, n_layer=1)
    t.check(t.run(dev))


@pytest.mark.parametrize("ct", CACHE_TYPES)
@pytest.mark.parametrize("heads,kv,hd,n", [(8, 2, 128, 20), (4, 1, 64, 9), (16, 2, 256, 12)])
def test_tree_attention_ragged_drafts_and_rows_that_see_nothing(KV, dev, ct, heads, kv, hd, n):
    """Fewer drafted tokens than rows (none at all, in one sequence), bits of rows that are not drafted, and rows
    of no bits, which without a history see nothing."""
    t = Tree(KV, ct, n, [50, 0, 300, 0], heads, kv, hd, seed=hd + n, drafts=[n, n - 3, 1, 0])
    t.seen[:, :, n - 2:] = True
    t.seen[0, 2] = False
    t.seen[1, 1] = False
    t.check(t.run(dev))


@pytest.mark.parametrize("ct", CACHE_TYPES)
@pytest.mark.parametrize("n,hd", [(3, 128), (40, 128), (30, 64), (20, 256)])
@pytest.mark.parametrize("past,width", [(200, 11), (900, 50)])
def test_tree_attention_missing_pages_are_zero_rows(KV, dev, ct, n, hd, past, width):
    """Table entries of -1, and positions past the table's end, are keys of score 0 and value 0."""
    t = Tree(KV, ct, n, [past, 90], 8, 2, hd, seed=3, holes=[(0, 1), (0, 5), (1, 0)])
    t.tables = np.ascontiguousarray(t.tables[:, :width])
    empty = np.zeros((0, 2 * hd), np.float32)
    t.hist = [[KV.gather(ct, a, t.n_layer, t.layer, t.tables[b], p, empty).reshape(p, 2, hd) for a in t.arena]
              for b, p in enumerate(t.pasts)]
    t.check(t.run(dev))


@pytest.mark.parametrize("n,hd", [(3, 64), (40, 128), (24, 256)])
def test_tree_attention_of_q8_0_values_past_the_f16_range(KV, dev, n, hd):
    """Slots of magnitudes that no f16 piece holds, with queries as much smaller."""
    t = Tree(KV, Q8_0, n, [300, 20], 8, 2, hd, seed=hd, spread=2.0 ** 18, n_layer=1)
    t.q *= 2.0 ** -18
    t.check(t.run(dev))


def test_tree_attention_without_mask_is_a_chain(KV, dev):
    t = Tree(KV, F16, 70, [77, 0], 4, 2, 64, seed=5)
    t.seen[:] = np.tril(np.ones((70, 70), bool))
    out = t.cache(dev).tree_attention(*t.args(dev))
    t.check(to_host(out).reshape(2, 70, 4, 64))
    # n_past and the cached causal attention agree within both bounds
    one = t.cache(dev).attention(t.layer, to_dev(t.tables[0], dev), *(x[:70] for x in t.args(dev)[4:7]), 77, t.scale)
    assert np.allclose(to_host(one), to_host(out)[:70], rtol=0, atol=1e-5)


def test_tree_attention_past_is_clamped(KV, dev):
    """Lengths above max_past or below 0 count as max_past and 0; draft counts as 0 .. n_tokens."""
    t = Tree(KV, F16, 6, [90, 60], 8, 2, 64, seed=6)
    args = list(t.args(dev))
    args[2], args[3] = i32([1 << 30, -5], dev), 90
    out = t.cache(dev).tree_attention(*args, **{**t.kwargs(dev), "n_draft": i32([1000, -1], dev)})
    t.drafts, t.hist[1] = [6, 0], [x[:0] for x in t.hist[1]]
    t.check(to_host(out).reshape(2, 6, 8, 64))


@pytest.mark.parametrize("ct", CACHE_TYPES)
@pytest.mark.parametrize("n,heads,kv,hd", [(6, 8, 2, 128), (40, 8, 2, 128), (30, 4, 1, 64), (20, 8, 2, 256)])
@pytest.mark.parametrize("past", [200, 777])
def test_tree_attention_hidden_infinities_and_nan(KV, dev, ct, n, heads, kv, hd, past):
    """Drafted rows full of infinities and NaN reach only the rows that see them; a NaN beyond the drafted
    tokens reaches none."""
    t = Tree(KV, ct, n, [70, past], heads, kv, hd, seed=7, drafts=[n, n - 2])
    t.seen[:, 2:, 1] = False
    t.seen[:, :, 3] = False
    t.kc[:, 1], t.vc[:, 1] = np.nan, np.inf
    t.vc[:, 3, :, ::5] = -np.inf  # seen by no row
    t.kc[1, n - 2:], t.vc[1, n - 2:], t.q[1, n - 2:] = np.nan, np.nan, np.nan
    out = t.run(dev)
    assert np.isfinite(out[:, [0] + list(range(2, n - 2))]).all()
    t.check(out)


@pytest.mark.parametrize("ct", [F32, F16])
@pytest.mark.parametrize("n,heads,kv,hd", [(4, 8, 2, 128), (40, 8, 2, 128), (20, 8, 2, 64), (20, 8, 1, 256)])
@pytest.mark.parametrize("past", [150, 1100])
def test_tree_attention_infinities_in_the_cache(KV, dev, ct, n, heads, kv, hd, past):
    """As in the arithmetic of the definition: an infinite V element gives its dim that infinity, one of K a weight
    of 0 or NaN by the sign of the score, a NaN gives NaN."""
    t = Tree(KV, ct, n, [past], heads, kv, hd, seed=8, n_layer=1)
    dt = np.float32 if ct == F32 else np.float16
    k, v = (a.view(dt).reshape(t.n_blocks, 16, kv, hd) for a in t.arena)
    page = t.tables[0]
    v[page[2], 3, 0, 7] = np.inf
    k[page[4], 1, kv - 1, 5] = np.inf
    t.q[0, :n // 2, heads // kv * (kv - 1):, 5] = -np.abs(t.q[0, :n // 2, heads // kv * (kv - 1):, 5])  # scores of -inf
    empty = np.zeros((0, kv * hd), np.float32)
    t.hist = [[KV.gather(ct, a, 1, 0, page, past, empty).reshape(past, kv, hd) for a in t.arena]]
    out = t.run(dev)
    with np.errstate(invalid="ignore"):
        ref = S.tree_attention(t.q[0], *t.hist[0], t.kc[0], t.vc[0], t.seen[0], t.scale)[0]
    # a weight of exactly 0 beside an infinite value is NaN in 64 bits' underflow only; compare where both are finite
    assert np.array_equal(np.isinf(out[0]), np.isinf(ref)) and np.array_equal(np.isnan(out[0]), np.isnan(ref))
    ok = np.isfinite(ref)
    assert np.allclose(out[0][ok], ref[ok], rtol=1e-4, atol=1e-5)


@pytest.mark.parametrize("ct", CACHE_TYPES)
@pytest.mark.parametrize("n,hd", [(3, 128), (40, 64), (40, 128), (20, 256)])
def test_tree_attention_wide_values(KV, dev, ct, n, hd):
    """Rows whose magnitudes lie far apart: queries over 2^40, keys and values over 2^20 (F16: 2^12) octaves apart
    from key to key, and scores in the hundreds, so that a row's reference is raised many times."""
    t = Tree(KV, ct, n, [400], 8, 2, hd, seed=9, n_layer=1)
    rng = np.random.default_rng(10)
    t.q *= (2.0 ** rng.integers(-20, 5, (1, n, 8, 1))).astype(np.float32)
    span = 6 if ct == F16 else 10
    row = 2 * hd
    for x in range(2):
        rows = (rng.normal(size=(400, row)) * 2.0 ** rng.integers(-span, span // 2, (400, 1))).astype(np.float32)
        KV.write(ct, t.arena[x], 1, 0, t.tables[0], 0, rows)
    empty = np.zeros((0, row), np.float32)
    t.hist = [[KV.gather(ct, a, 1, 0, t.tables[0], 400, empty).reshape(400, 2, hd) for a in t.arena]]
    t.check(t.run(dev))


def planted(KV, ct, n, hd, scores, zero, seed, heads=8, kv=2):
    """A call whose cached keys have the given scores (in base 2, one sequence each) for every row, and values of
    zero at the positions `zero`; no row sees a drafted key."""
    t = Tree(KV, ct, n, [len(s) for s in scores], heads, kv, hd, seed=seed, n_layer=1)
    t.q[:] = 0
    t.q[..., 0] = 8 / (t.scale * np.log2(np.e))
    t.seen[:] = False
    empty = np.zeros((0, kv * hd), np.float32)
    for b, s in enumerate(scores):
        k = np.zeros((len(s), kv, hd), np.float32)
        k[:, :, 0] = np.asarray(s)[:, None] / 8
        v = t.rng.normal(size=k.shape).astype(np.float32) + 1
        v[zero] = 0
        for x, rows in enumerate((k, v)):
            KV.write(ct, t.arena[x], 1, 0, t.tables[b], 0, rows.reshape(len(s), -1))
    t.hist = [[KV.gather(ct, a, 1, 0, t.tables[b], p, empty).reshape(p, kv, hd) for a in t.arena]
              for b, p in enumerate(t.pasts)]
    return t


@pytest.mark.parametrize("ct", CACHE_TYPES)
@pytest.mark.parametrize("n,hd", [(40, 64), (40, 128), (40, 256), (3, 128)])
@pytest.mark.parametrize("jump", [12, 17, 24])
def test_tree_attention_a_key_far_above_those_beside_it(KV, dev, ct, n, hd, jump):
    """Scores that rise by less than what raises a row's reference, then a key far above them a few places on, of
    value zero: what the keys before it give must not be lost when the reference follows it."""
    s = np.full(320, -40.0)
    s[:64], s[64:96], s[100] = -8, 0, jump
    planted(KV, ct, n, hd, [s], [100], seed=hd + jump).run_and_check(dev)


@pytest.mark.parametrize("ct", CACHE_TYPES)
@pytest.mark.parametrize("n,hd", [(1, 64), (1, 128), (1, 256), (40, 64), (40, 128), (40, 256)])
@pytest.mark.parametrize("sink", [15, 24, 36, 60, 100])
def test_tree_attention_sinks(KV, dev, ct, n, hd, sink):
    """A first key far above the others whose value is zero: the output is the others', each of a weight far below
    the row's largest, in all of fp32's digits. In the second sequence the others' scores lie apart as well."""
    s = [np.zeros(600), np.random.default_rng(sink).uniform(-30, 0, 290)]
    s[0][0], s[1][0] = sink, sink
    planted(KV, ct, n, hd, s, [0], seed=hd + sink).run_and_check(dev)


OTHER_WIDTHS = {
    "random": lambda KV, dev, ct, hd: test_tree_attention(KV, dev, ct, 100, [700, 5, 333], 8, 2, hd),
    "far above": lambda KV, dev, ct, hd: [
        test_tree_attention_a_key_far_above_those_beside_it(KV, dev, ct, 100, hd, jump) for jump in (17, 24)],
    "sinks": lambda KV, dev, ct, hd: [test_tree_attention_sinks(KV, dev, ct, 100, hd, sink) for sink in (24, 60)],
    "hidden": lambda KV, dev, ct, hd: test_tree_attention_hidden_infinities_and_nan(KV, dev, ct, 100, 8, 2, hd, 777),
    "cached": lambda KV, dev, ct, hd: ct != Q8_0 and test_tree_attention_infinities_in_the_cache(
        KV, dev, ct, 100, 8, 2, hd, 600),
    "wide": lambda KV, dev, ct, hd: test_tree_attention_wide_values(KV, dev, ct, 100, hd),
    "missing pages": lambda KV, dev, ct, hd: test_tree_attention_missing_pages_are_zero_rows(KV, dev, ct, 100, hd, 900, 50),
    "several": lambda KV, dev, ct, hd: test_tree_attention(KV, dev, ct, 40 if hd == 256 else 20, [2001, 1030] * 8, 8, 2, hd),
}


@pytest.mark.parametrize("ct", CACHE_TYPES)
@pytest.mark.parametrize("hd", [64, 256])
@pytest.mark.parametrize("what", OTHER_WIDTHS)
def test_tree_attention_many_rows_at_other_widths(KV, dev, ct, hd, what):
    """400 rows of a KV head, or 160 and 80 of several sequences: as many as share their keys through blocks at head_dim
    64 and 256."""
    OTHER_WIDTHS[what](KV, dev, ct, hd)


def test_tree_attention_strided_rows_and_another_stream(KV, dev):
    """Rows of q, K / V, out and the tables inside wider tensors, on a stream other than the current one."""
    import torch
    t = Tree(KV, Q8_0, 9, [130, 300], 8, 2, 64, seed=11)
    layer, tables, past, max_past, q, kc, vc, scale = t.args(dev)

    def wide(x, extra):
        w = torch.full((x.shape[0], x.shape[1] + extra), 77, dtype=x.dtype, device=dev)
        w[:, :x.shape[1]] = x
        return w[:, :x.shape[1]]
    out = torch.full((18, 8 * 64 + 3), 5.0, device=dev)
    cache, kw = t.cache(dev), t.kwargs(dev)
    s = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(s):
        cache.tree_attention(layer, wide(tables, 5), past, max_past, wide(q, 4), wide(kc, 8), wide(vc, 8), scale,
                             out=out[:, :512], **kw)
    s.synchronize()
    t.check(to_host(out[:, :512]).reshape(2, 9, 8, 64))
    assert (to_host(out[:, 512:]) == 5.0).all()


def test_tree_attention_offsets_past_32_bits(KV, dev):
    """Pages beyond 4 GiB of an arena (made on the device; only the pages used are written)."""
    import torch
    n_blocks, kv, hd, past = 36000, 8, 256, 70
    cache = dc.PagedKVCache(F32, 1, 1, kv, hd, device=dev)
    page = 16 * kv * hd * 4
    assert n_blocks * page > 1 << 32
    cache.n_blocks = n_blocks
    cache.k, cache.v = (torch.empty(n_blocks * page, dtype=torch.uint8, device=dev) for _ in range(2))
    table = np.array([35999, 3, 34000, 33500, 35000], np.int32)
    rng = np.random.default_rng(12)
    hist = [rng.normal(size=(past, kv * hd)).astype(np.float32) for _ in range(2)]
    for which, rows in zip("kv", hist):
        cache.write(which, 0, i32(table, dev), 0, to_dev(rows, dev))
    q = rng.normal(size=(2, 8, hd)).astype(np.float32)
    kc, vc = (rng.normal(size=(2, kv, hd)).astype(np.float32) for _ in range(2))
    out = cache.tree_attention(0, i32(table[None], dev), i32([past], dev), past, to_dev(q.reshape(2, -1), dev),
                               to_dev(kc.reshape(2, -1), dev), to_dev(vc.reshape(2, -1), dev), 0.0625)
    ref = S.tree_attention(q, *(x.reshape(past, kv, hd) for x in hist), kc, vc, np.tril(np.ones((2, 2), bool)), 0.0625)[0]
    assert np.allclose(to_host(out).reshape(2, 8, hd), ref, rtol=0, atol=2e-5)


@pytest.mark.parametrize("n,pasts", [(7, [100]), (24, [3000, 700]), (64, [2000])])
def test_tree_attention_repeats_bit_for_bit_in_graphs(KV, dev, n, pasts):
    import torch
    t = Tree(KV, F16, n, pasts, 8, 2, 128, seed=13)
    cache, args, kw = t.cache(dev), t.args(dev), t.kwargs(dev)
    out = torch.empty_like(args[4])
    need = dc.kv_tree_attention_workspace_size(8, 2, 128, t.s, n, max(pasts))
    kw["workspace"] = torch.empty(max(need, 256), dtype=torch.uint8, device=dev)
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        cache.tree_attention(*args, out=out, **kw)
    torch.cuda.synchronize()
    want = out.clone()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        cache.tree_attention(*args, out=out, **kw)
    for _ in range(3):
        out.fill_(float("nan"))
        kw["workspace"].fill_(255)
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)


# ---------------------------------------------------------------- accepted paths
@pytest.mark.parametrize("ct", CACHE_TYPES)
@pytest.mark.parametrize("kv,hd", [(2, 64), (8, 128), (1, 256)])
def test_write_path_bytes(KV, dev, ct, kv, hd):
    rng = np.random.default_rng(20 + hd)
    n_layer, n_blocks, s, n, p, row = 3, 12, 4, 6, 5, kv * hd
    tables = np.full((s, 4), -1, np.int32)
    tables[:3, :3] = rng.permutation(n_blocks)[:9].reshape(3, 3)
    tables[3] = [n_blocks + 5, 2000000000, -7, -1]  # no pages
    past, n_path = [14, 0, 45, 3], [5, 3, 5, 5]     # over a page's end; the third past the pages it has
    path = np.array([[0, 2, 3, 5, 4], [1, -1, 6, 0, 0], [5, 4, 3, 2, 1], [0, 1, 2, 3, 4]], np.int32)
    cur = [rng.normal(size=(n_layer, s, n, row)).astype(np.float32) for _ in range(2)]
    cache = dc.PagedKVCache(ct, n_blocks, n_layer, kv, hd, device=dev)
    start = [rng.integers(0, 255, cache.k.numel(), dtype=np.uint8) for _ in range(2)]
    cache.k.copy_(to_dev(start[0], dev))
    cache.v.copy_(to_dev(start[1], dev))
    cache.write_path(i32(tables, dev), i32(past, dev), i32(path, dev), i32(n_path, dev),
                     *(to_dev(x.reshape(n_layer, s * n, row), dev) for x in cur))
    for arena, x, got in zip(start, cur, (cache.k, cache.v)):
        S.write_path(ct, arena, n_blocks, n_layer, tables, past, path, n_path, x)
        assert np.array_equal(to_host(got), arena)
    # all places of every path, from the rows of wider tensors
    wide = [to_dev(np.concatenate([x, x], -1).reshape(n_layer, s * n, 2 * row), dev)[:, :, :row] for x in cur]
    cache.write_path(i32(tables, dev), i32(past, dev), i32(path, dev), None, *wide)
    for arena, x, got in zip(start, cur, (cache.k, cache.v)):
        S.write_path(ct, arena, n_blocks, n_layer, tables, past, path, [p] * s, x)
        assert np.array_equal(to_host(got), arena)


# ---------------------------------------------------------------- forks and compaction
def filled_cache(ct, n_blocks, n_layer, kv, hd, dev, seed):
    cache = dc.PagedKVCache(ct, n_blocks, n_layer, kv, hd, device=dev)
    rng = np.random.default_rng(seed)
    start = [rng.integers(0, 255, cache.k.numel(), dtype=np.uint8) for _ in range(2)]
    cache.k.copy_(to_dev(start[0], dev))
    cache.v.copy_(to_dev(start[1], dev))
    return cache, start


def assert_pages(cache, start, pairs):
    for got, arena in zip((cache.k, cache.v), start):
        want = arena.reshape(cache.n_blocks, -1).copy()
        for src, dst in pairs:
            want[dst] = arena.reshape(cache.n_blocks, -1)[src]
        assert np.array_equal(to_host(got).reshape(want.shape), want)


def check_fork(cache, start, tables, lengths, parents, refs, dev):
    want = S.fork([list(map(int, t)) for t in tables], list(lengths), list(parents), list(refs))
    got = cache.fork(i32(tables, dev), i32(lengths, dev), i32(parents, dev), i32(refs, dev))
    for name, g, w in zip(("tables", "lengths", "refs", "missing"), got, want[:3] + ([want[3]],)):
        assert np.array_equal(to_host(g), np.array(w)), name
    assert_pages(cache, start, want[4])
    return want


FORKS = [
    # (requests, beams, pages of a shared prompt, free pages, pages of the arena beyond all of them)
    (1, 1, 0, 2, 0), (1, 4, 9, 6, 0), (3, 5, 2, 4, 3), (16, 8, 14, 130, 0),
    (2, 8, 3, 1, 0),            # too few free pages
    (5, 6, 40, 40, 1500),       # several steps of the search for free pages
    (7, 9, 300, 70, 20000),     # the counts in device memory
]


@pytest.mark.parametrize("ct,kv,hd,n_layer", [(F16, 1, 64, 2), (Q8_0, 1, 32, 1), (F32, 2, 64, 3)])
@pytest.mark.parametrize("batch,beams,prefix,free,extra", FORKS)
def test_fork(dev, ct, kv, hd, n_layer, batch, beams, prefix, free, extra):
    rng = np.random.default_rng(batch + beams + prefix)
    n_blocks = batch * (prefix + 2 * beams) + free + extra
    cache, start = filled_cache(ct, n_blocks, n_layer, kv, hd, dev, 30)
    order, at, tables, lengths = rng.permutation(n_blocks), 0, [], []
    refs = np.zeros(n_blocks, np.int64)
    for _ in range(batch):
        shared = order[at:at + prefix]
        at += prefix
        for _ in range(beams):
            own = order[at:at + 2]
            at += 2
            full = rng.random() < 0.2
            tables.append(list(shared) + list(own))
            lengths.append((prefix + 2) * 16 if full else (prefix + 1) * 16 + int(rng.integers(1, 16)))
            np.add.at(refs, tables[-1], 1)
    refs[order[len(order) - extra:]] += extra > 0  # pages of others
    parents = np.concatenate([i * beams + rng.integers(0, beams, beams) for i in range(batch)])
    check_fork(cache, start, tables, lengths, parents, refs, dev)


def test_fork_parents_lengths_and_holders_out_of_the_ordinary(dev):
    """Parents that are none, empty sequences, lengths past the table, entries that are no pages, a partial page
    shared by two sequences, by one beyond the call, or that is a full page of another."""
    cache, start = filled_cache(F16, 40, 2, 1, 64, dev, 31)
    tables = [[3, 5, 7, -1], [3, 5, 9, -1], [4, 8, -1, -1], [10, 11, 12, 13], [-1, 50, 14, -1], [20, 21, 8, 2], [15, 40, -1, -1]]
    lengths = [40, 33, 20, 64, 37, 60, 24]
    refs = np.zeros(40, np.int64)
    for t, n in zip(tables, lengths):
        for p in t[:-(-n // 16)]:
            if 0 <= p < 40:
                refs[p] += 1
    refs[[7, 30]] += 1  # held beyond the call too
    for parents in ([0, 1, 2, 3, 4, 5, 6], [0, 0, 1, 1, 2, 2, 5, 5], [-1, 7, 1 << 30, 4, 4, 6, 6], [3] * 9, [2, 5]):
        check_fork(cache, start, tables, lengths, parents, refs, dev)
        cache, start = filled_cache(F16, 40, 2, 1, 64, dev, 32)
    check_fork(cache, start, tables, [0, -5, 1 << 30, 64, 0, 0, 0], [0, 1, 2, 2, 3, 3], refs, dev)


@pytest.mark.parametrize("n_blocks", [40, 20000])
def test_fork_counts_that_are_too_low(dev, n_blocks):
    """Pages that children hold though the counts say that nobody does are not taken as free: no page is the source
    and the target of copies, and the counts are the same from run to run."""
    tables = [[3, 0, 1, -1], [3, 0, 1, -1], [3, 5, 2, -1], [4, 6, 7, 8]]
    lengths = [40, 40, 37, 60]
    for low in (0, -1):
        refs = np.full(n_blocks, 1, np.int64)
        refs[[0, 1, 2, 3, 4, 5, 6, 7, 8, 11, 30, 31]] = low
        for parents in ([0], [0, 0], [0, 2, 2, 3, 3], [3, 3, 3, 0, 2, 0], [2, 2, 2, 2]):
            for _ in range(2):
                cache, start = filled_cache(F16, n_blocks, 1, 1, 64, dev, 37)
                check_fork(cache, start, tables, lengths, parents, refs, dev)


def test_fork_then_fork_again_leaves_no_page_behind(dev):
    """A beam search's forks one after another, each with the last one's tables and counts."""
    rng = np.random.default_rng(33)
    cache, start = filled_cache(F32, 24, 1, 1, 64, dev, 34)
    tables, lengths, refs = [[0, 1]] * 1, [24], [1, 1] + [0] * 22
    tables, lengths, refs, missing, pairs = check_fork(cache, start, tables, lengths, [0] * 4, refs, dev)
    for _ in range(6):
        start = [to_host(x) for x in (cache.k, cache.v)]
        parents = rng.integers(0, 4, 4)
        tables, lengths, refs, missing, pairs = check_fork(cache, start, tables, lengths, parents, refs, dev)
        assert missing == 0 and sum(refs) == 8 and sum(r > 0 for r in refs) == 5


@pytest.mark.parametrize("ct,kv,hd,n_layer", [(F16, 1, 64, 2), (Q8_0, 1, 32, 1), (F32, 4, 128, 3)])
@pytest.mark.parametrize("n_blocks,live", [(1, 1), (2, 1), (8, 0), (8, 8), (9, 4), (120, 70), (501, 250), (1024, 1023),
                                           (3000, 1500), (2500, 30)])
def test_compact(dev, ct, kv, hd, n_layer, n_blocks, live):
    rng = np.random.default_rng(n_blocks + live)
    cache, start = filled_cache(ct, n_blocks, n_layer, kv, hd, dev, 35)
    refs = np.zeros(n_blocks, np.int64)
    held = rng.permutation(n_blocks)[:live]
    refs[held] = rng.integers(1, 4, live)
    refs[rng.permutation(np.flatnonzero(refs == 0))[:2]] = -1  # counts below 0 are free pages
    tables = np.full((3, max(-(-live // 2), 1)), -1)
    tables[0, :len(held[::2])] = held[::2]
    tables[1, :len(held[1::2])] = held[1::2]
    tables[2, 0] = n_blocks + 7
    lengths = [16 * len(held[::2]), max(16 * len(held[1::2]) - 5, 0), 16]
    if live > 4:
        lengths[0] -= 32  # its last two entries hold nothing and keep their numbers
        refs[tables[0, len(held[::2]) - 2:len(held[::2])]] = 0
    t, r, n, pairs = S.compact(tables.tolist(), lengths, refs.tolist())
    got = cache.compact(i32(tables, dev), i32(lengths, dev), i32(refs, dev))
    assert np.array_equal(to_host(got[0]), t) and np.array_equal(to_host(got[1]), r) and int(to_host(got[2])[0]) == n
    assert_pages(cache, start, pairs)


@pytest.mark.parametrize("n_blocks,live", [(2049, 1000), (2050, 1025), (16000, 8000), (40000, 21000), (33000, 40)])
def test_compact_of_many_pages(dev, n_blocks, live):
    """Beyond the copies that are made beside the plan."""
    test_compact(dev, Q8_0, 1, 32, 1, n_blocks, live)


def test_memory_of_a_call_is_its_streams(KV, dev, monkeypatch):
    """Outputs and workspaces that a call on another stream makes come from that stream's memory."""
    import torch
    t = Tree(KV, F16, 3, [900, 40], 4, 2, 64, seed=9)
    cache, args = t.cache(dev), t.args(dev)
    refs = torch.zeros(t.n_blocks, dtype=torch.int32, device=dev)
    x, beam = torch.randn((2, 500), device=dev), torch.zeros((1, 2), device=dev)
    parents = i32([0, 1, 1], dev)
    kwargs = t.kwargs(dev)
    s = torch.cuda.Stream()
    torch.cuda.synchronize()
    made, empty = [], torch.empty

    def spy(*a, **kw):
        made.append(torch.cuda.current_stream().cuda_stream)
        return empty(*a, **kw)
    monkeypatch.setattr(torch, "empty", spy)
    out = cache.tree_attention(*args, **kwargs, stream=s.cuda_stream)
    forked = cache.fork(args[1], args[2], parents, refs, stream=s.cuda_stream)
    cache.compact(args[1], args[2], refs, stream=s.cuda_stream)
    dc.beam_select(x, beam, 2, stream=s.cuda_stream)
    assert len(made) == 15 and set(made) == {s.cuda_stream}
    assert torch.cuda.current_stream().cuda_stream != s.cuda_stream
    made.clear()
    dc.beam_select(x, beam, 2)
    assert set(made) == {torch.cuda.current_stream().cuda_stream}
    t.check(to_host(out).reshape(2, 3, 4, 64))
    assert forked[0].shape[0] == 3


def test_pages_in_graphs_and_on_streams(dev):
    """A fork and a compaction captured, replayed on changed inputs, on a stream of their own."""
    import torch
    cache, start = filled_cache(F16, 64, 2, 1, 64, dev, 36)
    tables, lengths = i32([[0, 9, 20], [0, 9, 33]], dev), i32([40, 41], dev)
    refs = torch.zeros(64, dtype=torch.int32, device=dev)
    refs[[0, 9]], refs[[20, 33]] = 2, 1
    parents = i32([0, 1, 0], dev)
    outs = [torch.empty(x, dtype=torch.int32, device=dev) for x in ((3, 3), (3,), (64,), (1,), (3, 3), (64,), (1,))]
    ws = torch.empty(1 << 16, dtype=torch.uint8, device=dev)

    def step():
        cache.fork(tables, lengths, parents, refs, *outs[:4], workspace=ws)
        cache.compact(outs[0], outs[1], outs[2], *outs[4:], workspace=ws)
    s = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(s):
        step()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        step()
    for order in ([1, 1, 1], [0, 1, 0], [1, 0, 1]):
        cache.k.copy_(to_dev(start[0], dev))
        cache.v.copy_(to_dev(start[1], dev))
        parents.copy_(i32(order, dev))
        for o in outs:
            o.fill_(-9)
        ws.fill_(255)
        torch.cuda.synchronize()
        g.replay()
        t, n, r, missing, pairs = S.fork(to_host(tables).tolist(), [40, 41], order, to_host(refs).tolist())
        t2, r2, live, moves = S.compact(t, n, r)
        want = [a.reshape(64, -1).copy() for a in start]
        for a in want:
            for src, dst in pairs + moves:
                a[dst] = a[src]
        for got, w in zip(outs, (t, n, r, [missing], t2, r2, [live])):
            assert np.array_equal(to_host(got), np.array(w))
        for got, w in zip((cache.k, cache.v), want):
            assert np.array_equal(to_host(got).reshape(w.shape), w)


# ---------------------------------------------------------------- beams
def check_beams(x, beam, n_out, dev, **kw):
    """Parents and tokens exactly. A score is rounded to fp32 (2^-24 of it); its lse is off by the roundings of
    the exponentials' arguments, |x - max| 2^-23 each weighted by its share of the sum, the exponentials' own and
    the partial sums': below 2^-20."""
    import torch
    s, p, t = dc.beam_select(x if torch.is_tensor(x) else to_dev(x, dev), to_dev(beam, dev), n_out, **kw)
    ref, rp, rt = S.beam_select(to_host(x).astype(np.float64) if torch.is_tensor(x) else x, beam, n_out)
    s = to_host(s)
    assert np.array_equal(to_host(p), rp) and np.array_equal(to_host(t), rt)
    none = ref == -np.inf
    assert np.array_equal(s == -np.inf, none)
    assert (np.abs(s - ref)[~none] <= 2.0 ** -23 * np.abs(ref[~none]) + 2.0 ** -20).all()


BEAMS = [(1, 1, 1, 1), (1, 1, 50, 64), (2, 3, 7, 21), (3, 2, 63, 5), (1, 4, 2048, 8), (2, 8, 2049, 16), (1, 1, 4097, 64),
         (24, 8, 8191, 16), (5, 5, 32000, 10), (1, 4, 151936, 8), (9, 7, 128257, 14), (300, 2, 1000, 4), (2, 256, 300, 64)]


@pytest.mark.parametrize("dtype", [np.float32, np.float16])
@pytest.mark.parametrize("b,w,v,n", BEAMS)
def test_beam_select(dev, dtype, b, w, v, n):
    rng = np.random.default_rng(b + w + v + n)
    x = (rng.normal(size=(b * w, v)) * 3).astype(dtype)
    x[np.arange(b * w), rng.integers(0, v, b * w)] = 9.0
    if v > 40:
        x[:, ::7] = -np.inf
    check_beams(x, (-3 * rng.random((b, w))).astype(np.float32), n, dev)


@pytest.mark.parametrize("b,w,v,n", [(1, 4, 151936, 64), (2, 16, 40000, 33), (1, 16, 60000, 64), (3, 9, 50000, 32),
                                     (1, 200, 12000, 64), (1, 256, 270000, 3)])
def test_beam_select_of_many_candidates(dev, b, w, v, n):
    """More outputs than a quarter of the groups, more candidates than the join's registers hold, and more lists."""
    test_beam_select(dev, np.float16 if v > 200000 else np.float32, b, w, v, n)


@pytest.mark.parametrize("dtype", [np.float32, np.float16])
def test_beam_select_ties_go_to_the_lowest(dev, dtype):
    """Equal logits (all of a row, all of a chunk and more than are ranked at once, negative and positive zeros),
    equal beams, and falling rows, whose largest lie in few threads."""
    rng = np.random.default_rng(40)
    for v in (5, 300, 2500, 20000):
        check_beams(np.zeros((6, v), dtype), np.zeros((2, 3), np.float32), 16, dev)
        x = rng.integers(0, 2, (6, v)).astype(dtype)
        x[0, ::2] *= -0.0
        check_beams(x, np.array([[0, -0.5, 0], [-1, -1, -1]], np.float32), 64, dev)
        fall = np.sort(rng.normal(size=v))[::-1].astype(dtype)
        check_beams(np.stack([fall, fall, fall[::-1], fall]), np.zeros((2, 2), np.float32), 33, dev)


def test_beam_select_rows_and_beams_without_continuations(dev):
    rng = np.random.default_rng(41)
    x = rng.normal(size=(12, 3000)).astype(np.float32)
    x[0, 77] = np.nan
    x[1, 5] = np.inf
    x[2] = -np.inf
    x[3, 10:] = -np.inf
    x[6:] = -np.inf
    x[7, 2999] = 4.0
    x[8, [0, 1500]] = 2.0
    x[9:] = np.nan
    beam = np.zeros((4, 3), np.float32)
    beam[1] = [np.nan, -np.inf, np.inf]
    x[4:6] = 1.0
    check_beams(x, beam, 20, dev)


def test_beam_select_strides_alignment_and_large_scores(dev):
    import torch
    rng = np.random.default_rng(42)
    for dtype in (torch.float32, torch.float16):
        base = (torch.randn(6 * 5007 + 64, device=dev) * 4).to(dtype)
        for off in (0, 1, 3, 5):
            x = base[off:off + 6 * 5007].view(6, 5007)[:, :4999]
            check_beams(x, (rng.random((2, 3)) * 10).astype(np.float32), 9, dev)
    # far from 0: sums must not overflow or vanish
    x = (rng.normal(size=(4, 700)) * 2000).astype(np.float32)
    check_beams(x, np.array([[-1e4, 1e4]] * 2, np.float32), 6, dev)


@pytest.mark.parametrize("low", [np.finfo(np.float32).min, np.float32(-3e38)])
def test_beam_select_masked_by_the_lowest_value(dev, low):
    """Tokens ruled out by the type's lowest value, as constrained decoding masks them: whole chunks of them beside
    ordinary ones, all but one token, and few enough others that the outputs reach them."""
    rng = np.random.default_rng(43)
    x = rng.normal(size=(6, 40000)).astype(np.float32)
    x[0, :9000] = low
    x[1, 8192:] = low
    x[2] = low
    x[2, 39999] = 1.5
    x[3] = low
    x[3, [5, 20000]] = 0.0
    x[4, 100:] = low
    check_beams(x, np.zeros((2, 3), np.float32), 8, dev)
    check_beams(x[[2]], np.zeros((1, 1), np.float32), 4, dev)
    check_beams(x[[3, 0], :700], np.array([[0, -2.0]], np.float32), 12, dev)


@pytest.mark.parametrize("v", [1, 700, 9000, 40000])
@pytest.mark.parametrize("value", [np.finfo(np.float32).min, np.finfo(np.float32).max, -3e38, 2.5e38, 1e12, -1e12])
def test_beam_select_rows_of_one_far_value(dev, v, value):
    """All of a row at a value from which its lse differs by less than a last bit, in 64 bits too: every score is the
    beam's less log v. Bound as in check_beams."""
    x = np.full((2, v), value, np.float32)
    s, p, t = (to_host(y) for y in dc.beam_select(to_dev(x, dev), to_dev(np.array([[-1.0, 2.0]], np.float32), dev), 5))
    n = min(v, 5)
    want = 2.0 - np.log(v)
    assert (p[0, :n] == 1).all() and t[0, :n].tolist() == list(range(n))
    assert (np.abs(s[0, :n] - want) <= 2.0 ** -23 * abs(want) + 2.0 ** -20).all()


@pytest.mark.parametrize("at", [5e4, 65504.0, -6e4, 1e5, -1e6, 8e6])
def test_beam_select_of_logits_far_from_zero(dev, at):
    """Rows around one far value each, F16 as far as it goes: the same bound, whatever the logits' size."""
    rng = np.random.default_rng(44)
    beam = -rng.random((2, 3)).astype(np.float32)
    x = (at + rng.normal(size=(6, 9001)) * 8).astype(np.float32)
    check_beams(x, beam, 8, dev)
    if abs(at) <= 65504:
        check_beams(np.clip(x * (1 - 1e-3 * np.arange(6)[:, None]), -65504, 65504).astype(np.float16), beam, 8, dev)


def test_beam_select_in_graphs(dev):
    import torch
    x = torch.randn((8, 30001), device=dev)
    beam = -torch.rand((2, 4), device=dev)
    outs = [torch.empty((2, 8), device=dev)] + [torch.empty((2, 8), dtype=torch.int32, device=dev) for _ in range(2)]
    ws = torch.empty(dc.beam_select_workspace_size(2, 4, 30001, 8), dtype=torch.uint8, device=dev)
    s = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(s):
        dc.beam_select(x, beam, 8, *outs, workspace=ws)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        dc.beam_select(x, beam, 8, *outs, workspace=ws)
    for _ in range(3):
        x.normal_()
        ws.fill_(255)
        torch.cuda.synchronize()
        want = dc.beam_select(x, beam, 8)
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        for o, w in zip(outs, want):
            assert torch.equal(o, w)


# ---------------------------------------------------------------- the operators together
def _example():
    import importlib.util
    import os
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "search_decode.py")
    spec = importlib.util.spec_from_file_location("search_decode", path)
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    return mod


def _whole(ex, model, cache_type, tokens):
    """Logits of a sequence run at once, without a cache."""
    import torch
    s = ex.Search(model, cache_type)
    logits, _, _ = model.forward(torch.tensor([tokens], device="cuda"), s.cache, s.tables, s.lengths, 0)
    return logits.double().cpu().numpy()


def test_search_example_beams_and_speculation(dev):
    """The example's beams, from forked pages, score what their sequences score when run at once without a cache,
    and its speculative steps take the tokens that one-by-one greedy decoding takes. The model's products are
    made in 64 bits here (the library's round the activations to 8 bits, where a last bit can decide a step of
    2^-7), and an F32 cache holds the rows unrounded, so that fp32 roundings alone tell the two apart."""
    import torch
    ex = _example()

    class Smooth(ex.Model):
        @staticmethod
        def _product(w, x):
            return (x.double() @ dc.dequantize_rows(dc.TYPE_Q8_0, w[0], w[1], w[2]).double().T.contiguous()).float()

        @staticmethod
        def _residual(w, x, r):
            return Smooth._product(w, x) + r
    model = Smooth(layers=2, vocab=500, seed=3)
    prompt = (torch.arange(21, device="cuda") * 13 % 500)[None]
    search = ex.Search(model, dc.TYPE_F32)
    out, scores, missing = search.beams(prompt, beams=5, steps=30)
    assert int(missing) == 0 and search.length == 21 + 29
    out, scores = to_host(out), to_host(scores)[0]
    assert (np.diff(scores) <= 0).all() and len({tuple(o) for o in out.tolist()}) == 5
    for o, s in zip(out.tolist(), scores):
        x = _whole(ex, model, dc.TYPE_F32, prompt[0].tolist() + o)[20:-1]
        lp = x - np.log(np.exp(x - x.max(1, keepdims=True)).sum(1, keepdims=True)) - x.max(1, keepdims=True)
        assert abs(lp[np.arange(30), o].sum() - s) < 2e-2, "a beam's pages are not its sequence's"
    held = to_host(search.refs)
    n_live = int(search.keep(2))
    assert n_live == 4 and (to_host(search.refs) == ([1] * 4 + [0] * 60)).all() and held.sum() >= 20
    text = prompt[0].tolist() + out[2].tolist()
    x = _whole(ex, model, dc.TYPE_F32, text)[-1]
    first = int(x.argmax())
    taken = search.speculate(text[-1], [first, (first + 1) % 500, 7], [0, 0, 1])
    assert taken[0] == first and len(taken) >= 2  # the drafted first token was right
    x = _whole(ex, model, dc.TYPE_F32, text + [first])[-1]
    assert taken[1] == int(x.argmax()) and search.length == 50 + len(taken)
