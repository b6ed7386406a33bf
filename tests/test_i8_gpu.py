"""Layers in 8-bit integers on the GPU against the 64-bit restatement (oracle/i8.py).

Bounds, u = 2^-24 (half a step of fp32): an exact sum becomes a product by three roundings (the sum's, two scales'),
so 3 u relative; a residual or bias adds one of the result. F16 outputs add half a step, 2^-11 relative or 2^-25.
silu(g) u: g has 3 u, e^-g what |g| 3 u makes of it and 2 u of its own, the sum one and the quotient two more, so silu has
(8 + 3 |g|) u, and with the other product (12 + 3 |g|) u. Below g = -88 e^-g is infinite in fp32 and the result -0, off by
less than 1e-36 |u|. Weighted sums: 3 u of each term and one of each of the k + 1 additions, of the terms' magnitudes."""
import math
import zlib

import numpy as np
import pytest
import torch

import densecore_amd as dc
from oracle import i8 as I

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


def rng(*key):
    return np.random.default_rng([zlib.crc32(k.encode()) if isinstance(k, str) else int(k) for k in key])


def gpu(a, dev):
    return torch.from_numpy(np.ascontiguousarray(a)).to(dev)


def strided(a, dev, extra):
    """The array on the GPU as the first columns of wider rows."""
    wide = torch.zeros((*a.shape[:-1], a.shape[-1] + extra), dtype=torch.from_numpy(a).dtype, device=dev)
    wide[..., :a.shape[-1]] = torch.from_numpy(a).to(dev)
    return wide[..., :a.shape[-1]]


def i8_rows(r, *shape):
    q = r.integers(-127, 128, shape, dtype=np.int8)
    return q, r.uniform(0.2, 1.5, shape[:-1]).astype(np.float32) * np.float32(0.01)


def hidden(r, m, k, half):
    x = r.standard_normal((m, k)).astype(np.float32)
    x[:, r.integers(0, k, max(k // 50, 1))] *= 30
    return x.astype(np.float16) if half else x


# ---------------------------------------------------------------- rows to int8, norms
WIDTHS = [16, 48, 512, 528, 1024, 2048, 2560, 4096, 4112, 8192, 9728, 16384, 16400, 40000]


@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("k", WIDTHS)
def test_quantize(dev, k, half):
    r = rng("quantize", k, half)
    x = hidden(r, 7, k, half)
    q, s = dc.quantize_i8(gpu(x, dev))
    qr, sr = I.quantize(x)
    assert (q.cpu().numpy() == qr).all()
    assert (s.cpu().numpy() == sr).all()


def test_quantize_steps_halves_and_extremes(dev):
    """Halves go to even, the largest is +-127, rows of tiny and huge values keep their steps."""
    x = np.zeros((6, 32), np.float32)
    x[0, :] = np.arange(32) - 16 + 0.5
    x[0, 0] = 127.0
    x[1, :] = 3.0e38
    x[1, 1] = -1.5e38
    x[2, :] = 1e-42  # below the normal range
    x[2, 3] = -3e-42
    x[3, 5] = -2.0
    x[5, :] = np.float32(1.0) / 3
    q, s = dc.quantize_i8(gpu(x, dev))
    qr, sr = I.quantize(x)
    assert (q.cpu().numpy() == qr).all() and (s.cpu().numpy() == sr).all()
    assert q[0, 1].item() == -14 and q[0, 2].item() == -14 and s[4].item() == 0 and (q[4] == 0).all()


@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("half", [False, True])
def test_rows_that_are_not_finite_show_it(dev, value, half):
    x = hidden(rng("bad", half), 5, 2560, half)
    x[2, 1777] = value
    q, s = dc.quantize_i8(gpu(x, dev))
    assert math.isnan(s[2].item()) and (q[2] == 0).all()
    qr, sr = I.quantize(x)
    ok = [0, 1, 3, 4]
    assert (q.cpu().numpy()[ok] == qr[ok]).all() and (s.cpu().numpy()[ok] == sr[ok]).all()
    w = np.ones(2560, np.float32)
    h, q, s = dc.rms_norm_i8(gpu(x, dev), gpu(w, dev), 1e-6, r=gpu(np.zeros((5, 2560), np.float32), dev))
    assert math.isnan(s[2].item()) and (q[2] == 0).all() and not math.isfinite(h[2, 1777].item())
    assert torch.isfinite(s[ok]).all()
    y = dc.mul_mat_i8(q[:4].contiguous(), s[:4].nan_to_num(1.0), q, s)
    assert torch.isnan(y[2]).all() and torch.isfinite(y[ok]).all()


@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("residual", ["none", "new", "in_place"])
@pytest.mark.parametrize("m,k", [(1, 2560), (3, 16), (5, 528), (130, 4096), (2, 4112), (9, 8192), (3, 16400), (2, 40000)])
def test_rms_norm(dev, m, k, residual, half):
    r = rng("norm", m, k, residual, half)
    x, w = hidden(r, m, k, half), (1 + 0.3 * r.standard_normal(k)).astype(np.float32)
    res = None if residual == "none" else 3 * hidden(r, m, k, False)
    rt = None if res is None else strided(res, dev, 16)
    y = torch.empty((m, k), device=dev)
    h, q, s = dc.rms_norm_i8(strided(x, dev, 8), gpu(w, dev), 1e-5, r=rt, h=rt if residual == "in_place" else None, y=y)
    hr, qr, sr, yr = I.rms_norm(x, w, 1e-5, res)
    if res is None:
        assert h is None
    else:
        assert (h.cpu().numpy() == hr).all()
        assert residual != "in_place" or h.data_ptr() == rt.data_ptr()
    assert (q.cpu().numpy() == qr).all()
    assert (np.abs(s.cpu().numpy() - sr) <= 1.001 * U * sr).all()
    assert (np.abs(y.cpu().numpy() - yr) <= 1.001 * U * np.abs(yr) + 2.0 ** -149).all()
    # the fp32 rows alone, and the int8 rows alone
    _, y2 = dc.rms_norm(strided(x, dev, 8), gpu(w, dev), 1e-5, r=None if res is None else gpu(res, dev))
    assert torch.equal(y, y2)


def test_rms_norm_of_zeros_and_of_values_whose_squares_overflow(dev):
    x = np.zeros((3, 2560), np.float32)
    x[1] = 1e30 * rng("huge").standard_normal(2560)
    x[2] = 1e-30 * rng("small").standard_normal(2560)
    w = np.ones(2560, np.float32)
    _, q, s = dc.rms_norm_i8(gpu(x, dev), gpu(w, dev), 1e-6)
    _, qr, sr, _ = I.rms_norm(x, w, 1e-6)
    assert (q.cpu().numpy() == qr).all() and (np.abs(s.cpu().numpy() - sr) <= 1.001 * U * sr).all()
    assert s[0].item() == 0


# ---------------------------------------------------------------- products
SHAPES = [(9, 4097, 512), (16, 8200, 640), (14, 9728, 560), (20, 9730, 528), (30, 14340, 528), (45, 4100, 1040), (48, 9728, 768), (48, 12000, 528),
          (60, 8192, 656), (61, 9999, 768), (126, 4096, 512), (55, 4610, 528), (61, 3600, 528), (5, 4090, 8208), (30, 4096, 8192),
          (37, 100, 80), (1, 1, 16), (1, 9728, 2560), (1, 33, 131056), (3, 65, 272), (5, 1000, 768), (16, 17, 4096), (17, 300, 528), (31, 2560, 1024),
          (33, 64, 2048), (48, 513, 1040), (61, 2560, 9728), (40, 65536, 80), (64, 129, 112), (65, 100, 256), (100, 2560, 1040), (90, 200, 5008), (128, 128, 128), (250, 64, 65536),
          (129, 257, 400), (200, 1111, 3088), (256, 2048, 2048), (300, 5000, 656), (513, 770, 144), (700, 9728, 2560),
          (1025, 4096, 2064), (2048, 8192, 2048), (4099, 1500, 272)]


def check_product(y, w, ws, x, xs, r=None, half=False):
    ref = I.mul_mat(w, ws, x, xs)
    bound = 3.01 * U * np.abs(ref)
    if r is not None:
        ref = ref + r
        bound += 1.01 * U * np.abs(ref)
    if half:
        bound += 2.0 ** -11 * np.abs(ref) * 1.01 + 2.0 ** -25
    err = np.abs(y.double().cpu().numpy() - ref)
    assert (err <= bound).all(), f"worst {np.max(err / np.maximum(bound, 1e-300))} of its bound"


@pytest.mark.parametrize("m,n,k", SHAPES)
def test_mul_mat(dev, m, n, k):
    r = rng("product", m, n, k)
    w, ws = i8_rows(r, n, k)
    x, xs = i8_rows(r, m, k)
    y = dc.mul_mat_i8(gpu(w, dev), gpu(ws, dev), gpu(x, dev), gpu(xs, dev))
    check_product(y, w, ws, x, xs)
    # the same bits without a workspace, and again
    none = torch.full((m, n), 7.0, device=dev)
    t = [gpu(a, dev) for a in (w, ws, x, xs)]
    status = dc.lib().dcq_mul_mat_i8(t[0].data_ptr(), t[1].data_ptr(), n, k, k, t[2].data_ptr(), t[3].data_ptr(), m, k, None, 0,
                                     0, none.data_ptr(), 4 * n, None, 0, None)
    torch.cuda.synchronize()
    assert status == 0 and torch.equal(y, none)


@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("add", ["none", "residual", "bias", "in_place"])
@pytest.mark.parametrize("m,n,k", [(1, 100, 2560), (13, 257, 272), (61, 512, 4096), (70, 130, 2064), (600, 1029, 656)])
def test_mul_mat_of_strided_rows_with_an_addend(dev, m, n, k, add, half):
    if add == "in_place" and half:
        pytest.skip("R is fp32")
    r = rng("added", m, n, k, add, half)
    w, ws = i8_rows(r, n, k)
    x, xs = i8_rows(r, m, k)
    res = None if add == "none" else r.standard_normal(n if add == "bias" else (m, n)).astype(np.float32)
    y = torch.full((m, n + 5), 7.0, dtype=torch.float16 if half else torch.float32, device=dev)
    if add == "in_place":
        y[:, :n] = gpu(res, dev)
    rt = None if add == "none" else y[:, :n] if add == "in_place" else gpu(res, dev) if add == "bias" else strided(res, dev, 3)
    out = dc.mul_mat_i8(strided(w, dev, 32), gpu(ws, dev), strided(x, dev, 16), gpu(xs, dev), r=rt, y=y[:, :n])
    assert out.data_ptr() == y.data_ptr()
    check_product(out, w, ws, x, xs, res, half)
    assert (y[:, n:] == 7).all()


@pytest.mark.parametrize("n,k", [(200, 9728), (4100, 4096), (9728, 528), (2048, 2064), (14336, 2048), (1030, 272)])
def test_mul_mat_bits_do_not_depend_on_the_batch(dev, n, k):
    """A row's result with a residual or a bias is the same bits whichever kernel, tile or split serves its batch."""
    r = rng("bits", n, k)
    w, ws = (gpu(a, dev) for a in i8_rows(r, n, k))
    x, xs = (gpu(a, dev) for a in i8_rows(r, 700, k))
    for add in (gpu(r.standard_normal((700, n)).astype(np.float32) * 50, dev), gpu(r.standard_normal(n).astype(np.float32) * 50, dev)):
        whole = dc.mul_mat_i8(w, ws, x, xs, r=add)
        for m in (1, 12, 16, 30, 40, 61, 100, 200, 400):
            part = dc.mul_mat_i8(w, ws, x[:m], xs[:m], r=add if add.ndim == 1 else add[:m])
            assert torch.equal(part, whole[:m]), m


@pytest.mark.parametrize("m", [1, 40, 300])
def test_mul_mat_sums_of_the_largest_values_are_exact(dev, m):
    k, n = 131056, 40
    w, x = np.full((n, k), -128, np.int8), np.full((m, k), -128, np.int8)
    w[1] = 127
    one = np.ones(max(m, n), np.float32)
    y = dc.mul_mat_i8(gpu(w, dev), gpu(one[:n], dev), gpu(x, dev), gpu(one[:m], dev))
    assert (y[:, 0] == 128.0 * 128 * k).all() and (y[:, 1] == float(np.float32(-128.0 * 127 * k))).all()


# ---------------------------------------------------------------- the router
def check_route(dev, logits, k, **kw):
    bias = kw.get("bias")
    got = dc.moe_route(gpu(logits, dev), k, **{**kw, **({} if bias is None else {"bias": gpu(bias, dev)})})
    ids, weights = (t.cpu().numpy() for t in got)
    ri, rw = I.route(logits, k, **kw)
    assert (ids == ri).all(), f"{(ids != ri).sum()} of {ids.size} differ"
    assert (np.abs(weights - rw) <= 1.001 * U * np.abs(rw) + 2.0 ** -149).all()
    return ids, weights


@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("m,e,k,groups,kept,best", [(1, 1, 1, 1, 1, 1), (5, 128, 8, 1, 1, 1), (33, 60, 4, 1, 1, 1), (70, 256, 8, 8, 4, 2),
                                                    (9, 160, 6, 8, 3, 1), (17, 512, 10, 1, 1, 1), (4, 64, 64, 64, 64, 2),
                                                    (40, 384, 6, 4, 2, 2), (3, 300, 33, 2, 1, 1)])
def test_route(dev, m, e, k, groups, kept, best, scoring, half):
    r = rng("route", m, e, k, scoring, half)
    x = (2 * r.standard_normal((m, e))).astype(np.float16 if half else np.float32)
    for bias in (None, (0.2 * r.standard_normal(e)).astype(np.float32)):
        for renorm in (True, False):
            check_route(dev, x, k, scoring=scoring, bias=bias, n_group=groups, topk_group=kept, group_best=best, renorm=renorm,
                        scale=2.5 if renorm else 1.0)


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
def test_route_ties_go_to_the_lower_expert(dev, scoring):
    x = np.zeros((4, 200), np.float32)
    x[1, 1::2] = 1
    x[2] = rng("ties").integers(0, 3, 200)
    x[3] = np.repeat(rng("ties", 1).integers(0, 4, 8), 25)
    for groups in (1, 8):
        check_route(dev, x, 9, scoring=scoring, n_group=groups, topk_group=max(groups // 2, 1), group_best=2)


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
def test_route_without_enough_experts(dev, scoring):
    """-infinity and biases that are not finite rule experts out; NaN and +infinity leave a token without any."""
    r = rng("few")
    x = r.standard_normal((9, 96)).astype(np.float32)
    x[0, 5:] = -np.inf
    x[1, :] = -np.inf
    x[2, 17] = np.nan
    x[3, 80] = np.inf
    x[4, :48] = -np.inf
    x[5, :] = np.finfo(np.float32).min
    x[6, :] = -3e4
    x[7, 3] = 3e38
    bias = r.standard_normal(96).astype(np.float32)
    check_route(dev, x, 8, scoring=scoring)
    check_route(dev, x, 8, scoring=scoring, n_group=6, topk_group=2, group_best=2)
    bias[[2, 3]] = np.inf, np.nan
    bias[10:16] = -np.inf
    ids, w = check_route(dev, x, 8, scoring=scoring, bias=bias, n_group=6, topk_group=2, group_best=2)
    assert not np.isin(ids, [2, 3, 10, 11, 12, 13, 14, 15]).any() and (ids[1:4] == -1).all() and (w[1:4] == 0).all()


def test_route_of_strided_rows(dev):
    x = rng("strided").standard_normal((21, 100)).astype(np.float32)
    ids, weights = dc.moe_route(strided(x, dev, 7), 5)
    ri, rw = I.route(x, 5)
    assert (ids.cpu().numpy() == ri).all() and np.allclose(weights.cpu().numpy(), rw, rtol=2 * U, atol=0)


# ---------------------------------------------------------------- experts
def experts(r, e, n, k):
    return i8_rows(r, e, n, k)


def some_ids(r, m, e, k, kind):
    if kind == "one":  # all tokens to the same experts
        return np.tile(r.permutation(e)[:k].astype(np.int32), (m, 1))
    if kind == "twice":  # one expert several times in a token
        return np.repeat(r.integers(0, e, (m, 1)), k, 1).astype(np.int32)
    ids = np.stack([r.permutation(e)[:k] for _ in range(m)]).astype(np.int32)
    if kind == "padded":
        ids[m // 2:] = -1
        ids[0, 0] = e
        ids[m // 4, -1] = -7
        ids[m // 3, 0] = 2 ** 31 - 1
    if kind == "none":
        ids[:] = -1
    return ids


EXPERTS = [(1, 8, 2, 64, 64, "mixed"), (5, 128, 8, 768, 2048, "mixed"), (1, 1, 1, 17, 16, "mixed"), (7, 16, 3, 100, 272, "padded"),
           (40, 4, 2, 130, 528, "padded"), (33, 8, 4, 65, 144, "one"), (20, 512, 6, 40, 80, "mixed"), (16, 3, 3, 48, 1040, "twice"),
           (9, 8, 2, 33, 64, "none"), (64, 16, 4, 96, 256, "mixed"), (150, 4, 2, 200, 400, "padded"), (300, 2, 2, 257, 144, "mixed"),
           (513, 8, 1, 64, 128, "mixed"), (700, 60, 4, 80, 160, "padded"), (1000, 3, 2, 300, 272, "mixed"), (260, 2, 2, 128, 2064, "one"),
           (60, 8, 4, 150, 528, "padded"), (130, 4, 1, 300, 1040, "mixed"), (1, 8, 2, 100, 4112, "mixed"), (3, 64, 4, 70, 144, "padded"),
           (1, 4, 1, 33, 1296, "mixed"), (900, 3, 2, 130, 272, "padded")]


@pytest.mark.parametrize("m,e,k,n,width,kind", EXPERTS)
def test_gate_up(dev, m, e, k, n, width, kind):
    r = rng("up", m, e, k, n, width)
    wg, wgs = experts(r, e, n, width)
    wu, wus = experts(r, e, n, width)
    x, xs = i8_rows(r, m, width)
    ids = some_ids(r, m, e, k, kind)
    h = torch.full((m * k, n + 3), 7.0, device=dev)
    plan = dc.moe_plan(gpu(ids, dev), e)
    args = (plan, gpu(wg, dev), gpu(wgs, dev), gpu(wu, dev), gpu(wus, dev), gpu(x, dev), gpu(xs, dev), k)
    dc.moe_gate_up_i8(*args, h=h[:, :n])
    ref, gate, up = I.gate_up(ids, e, wg, wgs, wu, wus, x, xs)
    bound = (12.1 + 3.01 * np.abs(gate)) * U * np.abs(ref) + 1e-36 * np.abs(up)
    got = h[:, :n].double().cpu().numpy()
    assert (np.abs(got - ref) <= bound).all()
    assert (h[:, n:] == 7).all()
    half = dc.moe_gate_up_i8(*args, dtype=torch.float16).double().cpu().numpy()
    lim = np.abs(ref) < 65000
    assert (np.abs(half - ref) <= bound + 2.0 ** -11 * 1.01 * np.abs(ref) + 2.0 ** -25)[lim].all()


@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("residual", ["none", "new", "in_place"])
@pytest.mark.parametrize("m,e,k,n,width,kind", EXPERTS)
def test_down(dev, m, e, k, n, width, kind, residual, half):
    if residual == "in_place" and half:
        pytest.skip("R is fp32")
    r = rng("down", m, e, k, n, width, residual)
    w, ws = experts(r, e, n, width)
    h, hs = i8_rows(r, m * k, width)
    ids = some_ids(r, m, e, k, kind)
    weights = r.uniform(0, 1, (m, k)).astype(np.float32)
    weights[ids < 0] = np.nan  # what is there for padding does not count
    hs[ids.reshape(-1) < 0] = np.nan
    res = None if residual == "none" else r.standard_normal((m, n)).astype(np.float32)
    y = torch.full((m, n + 3), 7.0, dtype=torch.float16 if half else torch.float32, device=dev)
    rt = None if res is None else gpu(res, dev)
    if residual == "in_place":
        y[:, :n] = rt
        rt = y[:, :n]
    plan = dc.moe_plan(gpu(ids, dev), e)
    dc.moe_down_i8(plan, gpu(w, dev), gpu(ws, dev), gpu(h, dev), gpu(hs, dev), gpu(weights, dev), r=rt, y=y[:, :n])
    ref, size = I.down(ids, e, w, ws, h, hs, weights, res)
    bound = (k + 4.1) * U * size
    if half:
        bound = bound + 2.0 ** -11 * 1.01 * np.abs(ref) + 2.0 ** -25
    assert (np.abs(y[:, :n].double().cpu().numpy() - ref) <= bound).all()
    assert (y[:, n:] == 7).all()


@pytest.mark.parametrize("m", [20, 150, 600, 2200])
def test_experts_of_large_matrices(dev, m):
    """Matrices of more than 8 MB, by tiles of every height: sampled tokens."""
    r = rng("large experts", m)
    e, k, n, width = 3, 2, 4100, 2064
    wg, wgs = experts(r, e, n, width)
    wu, wus = experts(r, e, n, width)
    x, xs = i8_rows(r, m, width)
    h, hs = i8_rows(r, m * k, width)
    ids = some_ids(r, m, e, k, "mixed")
    ids[m // 2] = -1
    weights = r.uniform(0, 1, (m, k)).astype(np.float32)
    plan = dc.moe_plan(gpu(ids, dev), e)
    up = dc.moe_gate_up_i8(plan, gpu(wg, dev), gpu(wgs, dev), gpu(wu, dev), gpu(wus, dev), gpu(x, dev), gpu(xs, dev), k)
    y = dc.moe_down_i8(plan, gpu(wg, dev), gpu(wgs, dev), gpu(h, dev), gpu(hs, dev), gpu(weights, dev))
    at = np.concatenate([[0, m // 2, m - 1], r.integers(0, m, 20)])
    slots = (at[:, None] * k + np.arange(k)).reshape(-1)
    ref, gate, lin = I.gate_up(ids[at], e, wg, wgs, wu, wus, x[at], xs[at])
    assert (np.abs(up.double().cpu().numpy()[slots] - ref) <= (12.1 + 3.01 * np.abs(gate)) * U * np.abs(ref) + 1e-36 * np.abs(lin)).all()
    ref, size = I.down(ids[at], e, wg, wgs, h[slots], hs[slots], weights[at], None)
    assert (np.abs(y.double().cpu().numpy()[at] - ref) <= (k + 4.1) * U * size).all()


@pytest.mark.parametrize("e,k,n,width", [(8, 2, 130, 272), (64, 4, 70, 1040), (3, 3, 257, 2064)])
def test_experts_bits_do_not_depend_on_the_batch(dev, e, k, n, width):
    """A token's H rows and Y are the same bits whichever kernel and tiles serve its batch."""
    r = rng("experts' bits", e, k, n)
    m = 900
    wg, wgs, wu, wus = (gpu(a, dev) for a in (*experts(r, e, n, width), *experts(r, e, n, width)))
    wd, wds = (gpu(a, dev) for a in experts(r, e, n, width))
    x, xs = (gpu(a, dev) for a in i8_rows(r, m, width))
    h, hs = (gpu(a, dev) for a in i8_rows(r, m * k, width))
    ids = gpu(some_ids(r, m, e, k, "mixed"), dev)
    weights, res = gpu(r.uniform(0, 1, (m, k)).astype(np.float32), dev), gpu(r.standard_normal((m, n)).astype(np.float32), dev)

    def both(m):
        plan = dc.moe_plan(ids[:m], e)
        up = dc.moe_gate_up_i8(plan, wg, wgs, wu, wus, x[:m], xs[:m], k)
        return up, dc.moe_down_i8(plan, wd, wds, h[:m * k], hs[:m * k], weights[:m], r=res[:m])
    whole = both(m)
    for part in (1, 2, 8, 30, 100, 300, 500):
        up, down = both(part)
        assert torch.equal(up, whole[0][:part * k]) and torch.equal(down, whole[1][:part]), part


@pytest.mark.parametrize("m,e,k", [(1, 1, 1), (5, 128, 8), (1000, 512, 7), (4097, 60, 4), (3, 7, 2)])
def test_plan(dev, m, e, k):
    r = rng("plan", m, e, k)
    ids = r.integers(-2, e + 2, (m, k)).astype(np.int32)
    plan = dc.moe_plan(gpu(ids, dev), e).view(torch.int32).cpu().numpy()
    slots = m * k
    flat = np.where((ids < 0) | (ids >= e), e, ids).reshape(-1)
    order_at = -(-(e + 2) // 64) * 64
    assert (plan[:e + 2] == np.concatenate([[0], np.cumsum(np.bincount(flat, minlength=e + 1))])).all()
    assert (plan[order_at:order_at + slots] == np.argsort(flat, kind="stable")).all()
    at = order_at + -(-slots // 64) * 64
    assert (plan[at:at + slots] == np.where(flat < e, flat, -1)).all()


# ---------------------------------------------------------------- the largest sizes
def spread_rows(a, dev, stride):
    """int8 rows as the first columns of rows `stride` bytes apart."""
    wide = torch.empty((len(a), stride), dtype=torch.int8, device=dev)
    wide[:, :a.shape[1]] = gpu(a, dev)
    return wide[:, :a.shape[1]]


@pytest.mark.parametrize("m,n,k", [(300, 290, 272), (40, 290, 272), (290, 9, 9728)])
def test_rows_of_the_largest_stride(dev, m, n, k):
    """2^24 bytes between rows: the last rows lie more than 2^32 bytes behind the first."""
    r = rng("spread", m, n, k)
    w, ws = i8_rows(r, n, k)
    x, xs = i8_rows(r, m, k)
    res = r.standard_normal((m, n)).astype(np.float32)
    wide = torch.empty((m, 1 << 22), device=dev)
    wide[:, :n] = gpu(res, dev)
    args = spread_rows(w, dev, 1 << 24), gpu(ws, dev), spread_rows(x, dev, 1 << 24), gpu(xs, dev)
    check_product(dc.mul_mat_i8(*args, r=wide[:, :n], y=wide[:, :n]), w, ws, x, xs, res)


def test_outputs_past_32_bits(dev):
    """Dense outputs of 5 GiB, and of experts 4.3: rows of every part of them."""
    r = rng("outputs")
    m, n, k = 41000, 32768, 32
    w, ws = i8_rows(r, n, k)
    x, xs = i8_rows(r, m, k)
    y = dc.mul_mat_i8(gpu(w, dev), gpu(ws, dev), gpu(x, dev), gpu(xs, dev))
    at = np.concatenate([[0, m - 1], r.integers(0, m, 60)])
    check_product(y[torch.from_numpy(at).to(dev)], w, ws, x[at], xs[at])
    del y
    m, e, top, n = 8200, 8, 4, 32768
    ids = some_ids(r, m, e, top, "mixed")
    wg, wgs = experts(r, e, n, k)
    wu, wus = experts(r, e, n, k)
    plan = dc.moe_plan(gpu(ids, dev), e)
    h = dc.moe_gate_up_i8(plan, gpu(wg, dev), gpu(wgs, dev), gpu(wu, dev), gpu(wus, dev), gpu(x[:m], dev), gpu(xs[:m], dev), top)
    assert h.numel() * 4 > 2 ** 32
    at = np.concatenate([[0, m - 1], r.integers(0, m, 20)])
    got = h.view(m, top, n)[torch.from_numpy(at).to(dev)].reshape(-1, n).double().cpu().numpy()
    ref, gate, up = I.gate_up(ids[at], e, wg, wgs, wu, wus, x[at], xs[at])
    assert (np.abs(got - ref) <= (12.1 + 3.01 * np.abs(gate)) * U * np.abs(ref) + 1e-36 * np.abs(up)).all()


@pytest.mark.parametrize("m", [1, 6, 60, 400])
def test_experts_far_apart(dev, m):
    """2^31 bytes and more between experts, 64 KiB between their rows."""
    r = rng("far", m)
    e, top, n, k = 4, 2, 40, 272
    ids = some_ids(r, m, e, top, "mixed")
    wg, wgs = experts(r, e, n, k)
    wu, wus = experts(r, e, n, k)
    room = torch.empty((2, e, (1 << 31) + 4096), dtype=torch.int8, device=dev)
    far = [t[:, :n << 16].unflatten(1, (n, 1 << 16))[..., :k] for t in room]
    for t, v in zip(far, (wg, wu)):
        t.copy_(gpu(v, dev))
    x, xs = i8_rows(r, m, k)
    plan = dc.moe_plan(gpu(ids, dev), e)
    h = dc.moe_gate_up_i8(plan, far[0], gpu(wgs, dev), far[1], gpu(wus, dev), gpu(x, dev), gpu(xs, dev), top).double().cpu().numpy()
    ref, gate, up = I.gate_up(ids, e, wg, wgs, wu, wus, x, xs)
    assert (np.abs(h - ref) <= (12.1 + 3.01 * np.abs(gate)) * U * np.abs(ref) + 1e-36 * np.abs(up)).all()
    hq, hs = i8_rows(r, m * top, k)
    weights = r.uniform(0, 1, (m, top)).astype(np.float32)
    y = dc.moe_down_i8(plan, far[1], gpu(wus, dev), gpu(hq, dev), gpu(hs, dev), gpu(weights, dev)).double().cpu().numpy()
    ref, size = I.down(ids, e, wu, wus, hq, hs, weights, None)
    assert (np.abs(y - ref) <= (top + 4.1) * U * size).all()


@pytest.mark.parametrize("m,e,k", [(1, 64, 16), (1, 64, 17), (2, 512, 16), (2, 512, 64), (16, 512, 16), (3, 40, 33)])
def test_many_experts_of_a_token(dev, m, e, k):
    """Up to 16 slots a token are a workgroup's waves; more go by the plan."""
    r = rng("many", m, e, k)
    n, width = 48, 528
    w, ws = experts(r, e, n, width)
    h, hs = i8_rows(r, m * k, width)
    ids = some_ids(r, m, e, k, "mixed")
    ids[0, k // 2] = -1
    weights = r.uniform(0, 1, (m, k)).astype(np.float32)
    plan = dc.moe_plan(gpu(ids, dev), e)
    y = dc.moe_down_i8(plan, gpu(w, dev), gpu(ws, dev), gpu(h, dev), gpu(hs, dev), gpu(weights, dev))
    ref, size = I.down(ids, e, w, ws, h, hs, weights, None)
    assert (np.abs(y.double().cpu().numpy() - ref) <= (k + 4.1) * U * size).all()


def test_the_largest_plan_and_routing(dev):
    """2^22 slots of 512 experts: the plan against a stable sort, the choices of sampled tokens against the oracle's."""
    r = rng("largest")
    m, e, k = 1 << 19, 512, 8
    g = torch.Generator(device=dev)
    g.manual_seed(5)
    logits = torch.randn((m, e), generator=g, device=dev, dtype=torch.float16)
    ids, weights = dc.moe_route(logits, k)
    at = np.concatenate([[0, m - 1], r.integers(0, m, 500)])
    ri, rw = I.route(logits[torch.from_numpy(at).to(dev)].cpu().numpy(), k)
    assert (ids.cpu().numpy()[at] == ri).all() and (np.abs(weights.cpu().numpy()[at] - rw) <= 1.001 * U * rw).all()
    plan = dc.moe_plan(ids, e).view(torch.int32)
    flat, order_at = ids.view(-1).long(), -(-(e + 2) // 64) * 64
    assert torch.equal(plan[order_at:order_at + m * k].long(), torch.sort(flat, stable=True).indices)
    assert torch.equal(plan[1:e + 1].long(), torch.cumsum(torch.bincount(flat, minlength=e), 0))


@pytest.mark.parametrize("half", [False, True])
def test_norm_of_rows_past_32_bits(dev, half):
    r = rng("norm rows", half)
    m, k = 300, 2560
    x, w = hidden(r, m, k, half), (1 + 0.3 * r.standard_normal(k)).astype(np.float32)
    wide = torch.empty((m, (1 << 24) // x.itemsize), dtype=torch.from_numpy(x).dtype, device=dev)
    wide[:, :k] = gpu(x, dev)
    q = torch.empty((m, 1 << 24), dtype=torch.int8, device=dev)[:, :k]
    _, q, s = dc.rms_norm_i8(wide[:, :k], gpu(w, dev), 1e-5, q=q)
    _, qr, sr, _ = I.rms_norm(x, w, 1e-5)
    assert (q.cpu().numpy() == qr).all() and (np.abs(s.cpu().numpy() - sr) <= 1.001 * U * sr).all()


# ---------------------------------------------------------------- the calls together, and how programs make them
def layer_inputs(dev, m, e=16, top=3, hidden=272, width=144, seed=0):
    g = torch.Generator(device=dev)
    g.manual_seed(seed)
    rnd = lambda *shape: torch.randn(shape, generator=g, device=dev)  # noqa: E731
    q = lambda *shape: tuple(t.view(*shape[:-1], *t.shape[1:]) for t in dc.quantize_i8(rnd(math.prod(shape[:-1]), shape[-1])))  # noqa: E731
    return {"x": rnd(m, hidden), "r": rnd(m, hidden), "w": rnd(hidden), "router": q(e, hidden), "gate": q(e, width, hidden),
            "up": q(e, width, hidden), "down": q(e, hidden, width), "top": top, "e": e}


def layer_buffers(dev, st):
    m, hidden = st["x"].shape
    e, width = st["gate"][0].shape[:2]
    new = lambda *shape, dtype=torch.float32: torch.zeros(shape, dtype=dtype, device=dev)  # noqa: E731
    return {"h": new(m, hidden), "q": new(m, hidden, dtype=torch.int8), "s": new(m), "logits": new(m, e),
            "ids": new(m, st["top"], dtype=torch.int32), "weights": new(m, st["top"]),
            "plan": new(dc.moe_plan_size(m, st["top"], e), dtype=torch.uint8), "g": new(m * st["top"], width),
            "gq": new(m * st["top"], width, dtype=torch.int8), "gs": new(m * st["top"]), "y": new(m, hidden),
            "ws": new(max(dc.moe_down_i8_workspace_size(m, st["top"], hidden), dc.mul_mat_i8_workspace_size(m, e, hidden), 256),
                      dtype=torch.uint8)}


def layer(st, b, stream=None):
    dc.rms_norm_i8(st["x"], st["w"], 1e-6, r=st["r"], h=b["h"], q=b["q"], s=b["s"], stream=stream)
    dc.mul_mat_i8(*st["router"], b["q"], b["s"], y=b["logits"], workspace=b["ws"], stream=stream)
    dc.moe_route(b["logits"], st["top"], ids=b["ids"], weights=b["weights"], stream=stream)
    dc.moe_plan(b["ids"], st["e"], plan=b["plan"], stream=stream)
    dc.moe_gate_up_i8(b["plan"], *st["gate"], *st["up"], b["q"], b["s"], st["top"], h=b["g"], stream=stream)
    dc.quantize_i8(b["g"], q=b["gq"], s=b["gs"], stream=stream)
    dc.moe_down_i8(b["plan"], *st["down"], b["gq"], b["gs"], b["weights"], r=b["h"], y=b["y"], workspace=b["ws"], stream=stream)
    return [b[n] for n in ("h", "q", "s", "logits", "ids", "weights", "g", "gq", "gs", "y")]


def check_layer(st, b):
    """Every stage against the oracle's of the stage before."""
    n = {k: v.cpu().numpy() for k, v in b.items()}
    host = {k: tuple(t.cpu().numpy() for t in v) for k, v in st.items() if isinstance(v, tuple)}
    h, q, s, _ = I.rms_norm(st["x"].cpu().numpy(), st["w"].cpu().numpy(), 1e-6, st["r"].cpu().numpy())
    assert (n["h"] == h).all() and (n["q"] == q).all() and (np.abs(n["s"] - s) <= 1.001 * U * s).all()
    check_product(b["logits"], *host["router"], n["q"], n["s"])
    ids, w = I.route(n["logits"], st["top"])
    assert (n["ids"] == ids).all() and (np.abs(n["weights"] - w) <= 1.001 * U * w).all()
    g, gate, up = I.gate_up(ids, st["e"], *host["gate"], *host["up"], n["q"], n["s"])
    assert (np.abs(n["g"] - g) <= (12.1 + 3.01 * np.abs(gate)) * U * np.abs(g) + 1e-36 * np.abs(up)).all()
    gq, gs = I.quantize(n["g"])
    assert (n["gq"] == gq).all() and (n["gs"] == gs).all()
    y, size = I.down(ids, st["e"], *host["down"], n["gq"], n["gs"], n["weights"], n["h"])
    assert (np.abs(n["y"] - y) <= (st["top"] + 4.1) * U * size).all()


@pytest.mark.parametrize("m", [1, 5, 70, 300])
def test_a_layer_of_all_calls(dev, m):
    st = layer_inputs(dev, m, seed=m)
    b = layer_buffers(dev, st)
    layer(st, b)
    check_layer(st, b)


@pytest.mark.parametrize("m", [1, 40, 130])
def test_graph_replays(dev, m):
    """Captured once, replayed on new inputs with eager work between: bit for bit the eager calls'."""
    st = layer_inputs(dev, m, seed=m)
    b, eager = layer_buffers(dev, st), layer_buffers(dev, st)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        layer(st, b)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        out = layer(st, b)
    for k in range(4):
        new = layer_inputs(dev, m, seed=100 + k)
        for name in ("x", "r"):
            st[name].copy_(new[name])
        for t in out:
            t.zero_()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for got, want in zip(out, layer(st, eager)):
            assert torch.equal(got, want)
        _ = torch.ones(1024, device=dev).sum().item()


def test_split_products_in_two_graphs_with_one_workspace(dev):
    """Replays one after the other: what a graph leaves in the workspace is no matter to the next."""
    r = rng("two graphs")
    m, n, k = 100, 200, 9728
    assert dc.mul_mat_i8_workspace_size(m, n, k) > 0
    ws = torch.full((dc.mul_mat_i8_workspace_size(m, n, k),), 85, dtype=torch.uint8, device=dev)
    sets = []
    for _ in range(2):
        w, x = i8_rows(r, n, k), i8_rows(r, m, k)
        args = [gpu(a, dev) for a in (*w, *x)]
        y = torch.zeros((m, n), device=dev)
        graph = torch.cuda.CUDAGraph()
        dc.mul_mat_i8(*args, y=y, workspace=ws)
        torch.cuda.synchronize()
        with torch.cuda.graph(graph):
            dc.mul_mat_i8(*args, y=y, workspace=ws)
        sets.append((graph, y, w, x, args))
    for _ in range(3):
        for graph, y, w, x, _ in sets:
            y.zero_()
            graph.replay()
        torch.cuda.synchronize()
        for _, y, w, x, _ in sets:
            check_product(y, *w, *x)


def test_two_streams_at_once(dev):
    """Two layers on streams of their own, buffers of their own: each its eager result."""
    sts = [layer_inputs(dev, m, seed=m) for m in (33, 90)]
    bufs = [layer_buffers(dev, st) for st in sts]
    want = [[t.clone() for t in layer(st, layer_buffers(dev, st))] for st in sts]
    streams = [torch.cuda.Stream() for _ in sts]
    torch.cuda.synchronize()
    for _ in range(5):
        outs = [layer(st, b, stream=s.cuda_stream) for st, b, s in zip(sts, bufs, streams)]
    torch.cuda.synchronize()
    for out, ref in zip(outs, want):
        assert all(torch.equal(a, b) for a, b in zip(out, ref))


def test_new_outputs_come_from_the_stream(dev):
    """Outputs and workspaces that a call makes for another stream: memory that the current one has just freed is not theirs."""
    r = rng("made")
    w, x = i8_rows(r, 300, 9728), i8_rows(r, 100, 9728)
    args = [gpu(a, dev) for a in (*w, *x)]
    stream = torch.cuda.Stream()
    torch.cuda.synchronize()
    for _ in range(3):
        y = dc.mul_mat_i8(*args, stream=stream.cuda_stream)
        torch.full((4 << 20,), 3.0, device=dev)  # freed at once, on the current stream
    stream.synchronize()
    check_product(y, *w, *x)


def test_a_plan_of_another_call_stays_inside_the_arrays(dev):
    """Wrong results, no access outside: numbers past the arrays' ends in every part of the plan."""
    st = layer_inputs(dev, 40, seed=3)
    b = layer_buffers(dev, st)
    layer(st, b)
    guard = torch.full((40 * st["top"] + 64, 144), 7.0, device=dev)
    h = guard[32:32 + 40 * st["top"]]
    for value in (0, -1, 7, 2 ** 31 - 1, -2 ** 31):
        b["plan"].view(torch.int32).fill_(value)
        dc.moe_gate_up_i8(b["plan"], *st["gate"], *st["up"], b["q"], b["s"], st["top"], h=h)
        dc.moe_down_i8(b["plan"], *st["down"], b["gq"], b["gs"], b["weights"], y=b["y"], workspace=b["ws"])
        torch.cuda.synchronize()
        assert (guard[:32] == 7).all() and (guard[-32:] == 7).all()


def test_padded_tokens_and_rows_behind_are_left(dev):
    """A batch padded with tokens of no expert: their H rows are zeros, their Y rows the residual; what lies behind stays."""
    st = layer_inputs(dev, 20, seed=9)
    b = layer_buffers(dev, st)
    layer(st, b)
    want = b["y"].clone()
    b["ids"][12:] = -1
    b["weights"][12:] = float("nan")
    b["gs"][12 * st["top"]:] = float("nan")
    dc.moe_plan(b["ids"], st["e"], plan=b["plan"])
    dc.moe_gate_up_i8(b["plan"], *st["gate"], *st["up"], b["q"], b["s"], st["top"], h=b["g"])
    assert (b["g"][12 * st["top"]:] == 0).all()
    wide = torch.full((22, 272), 7.0, device=dev)
    dc.moe_down_i8(b["plan"], *st["down"], b["gq"], b["gs"], b["weights"], r=b["h"], y=wide[:20], workspace=b["ws"])
    assert torch.equal(wide[:12], want[:12]) and torch.equal(wide[12:20], b["h"][12:]) and (wide[20:] == 7).all()


def test_binding_refusals(dev):
    r = rng("refused")
    w, ws = (gpu(a, dev) for a in i8_rows(r, 24, 64))
    x, xs = (gpu(a, dev) for a in i8_rows(r, 5, 64))
    f = torch.zeros((5, 64), device=dev)
    e3, e3s = w.view(1, 24, 64), ws.view(1, 24)
    plan = dc.moe_plan(torch.zeros((5, 1), dtype=torch.int32, device=dev), 1)
    for name, call in [
        ("w", lambda: dc.mul_mat_i8(w.float(), ws, x, xs)), ("x", lambda: dc.mul_mat_i8(w, ws, x[:, :48].t(), xs)),
        ("x", lambda: dc.mul_mat_i8(w, ws, x[:, :48], xs)), ("ws", lambda: dc.mul_mat_i8(w, ws[:20], x, xs)),
        ("xs", lambda: dc.mul_mat_i8(w, ws, x, xs.double())), ("y", lambda: dc.mul_mat_i8(w, ws, x, xs, y=f)),
        ("dtype", lambda: dc.mul_mat_i8(w, ws, x, xs, dtype=torch.bfloat16)), ("r", lambda: dc.mul_mat_i8(w, ws, x, xs, r=f)),
        ("r", lambda: dc.mul_mat_i8(w, ws, x, xs, r=ws.half())), ("ws", lambda: dc.mul_mat_i8(w, ws.cpu(), x, xs)),
        ("x", lambda: dc.quantize_i8(f.double())), ("q", lambda: dc.quantize_i8(f, q=f)), ("s", lambda: dc.quantize_i8(f, s=ws)),
        ("h", lambda: dc.rms_norm_i8(f, torch.ones(64, device=dev), 1e-6, h=f)), ("w", lambda: dc.rms_norm_i8(f, f[0, :32], 1e-6)),
        ("scoring", lambda: dc.moe_route(f, 2, scoring="tanh")), ("bias", lambda: dc.moe_route(f, 2, bias=ws)),
        ("ids", lambda: dc.moe_route(f, 2, ids=torch.zeros((5, 2), device=dev))), ("ids", lambda: dc.moe_plan(f, 2)),
        ("wu", lambda: dc.moe_gate_up_i8(plan, e3, e3s, e3[:, :12], e3s[:, :12].contiguous(), x, xs, 1)),
        ("wgs", lambda: dc.moe_gate_up_i8(plan, e3, ws, e3, e3s, x, xs, 1)), ("h", lambda: dc.moe_gate_up_i8(plan, e3, e3s, e3, e3s, x, xs, 1, h=f)),
        ("w", lambda: dc.moe_down_i8(plan, w, e3s, x, xs, f[:, :1])), ("weights", lambda: dc.moe_down_i8(plan, e3, e3s, x, xs, f[:, :1])),
        ("h", lambda: dc.moe_down_i8(plan, e3, e3s, x.float(), xs, f[:, :1].contiguous())),
    ]:
        with pytest.raises(ValueError, match=name):
            call()
    for call in (lambda: dc.moe_gate_up_i8(plan[:256], e3, e3s, e3, e3s, x, xs, 1), lambda: dc.mul_mat_i8(w, ws, x, xs, y=ws.expand(5, 24)[:5]),
                 lambda: dc.moe_route(f, 65), lambda: dc.rms_norm_i8(f, torch.ones(64, device=dev), -1.0),
                 lambda: dc.quantize_i8(torch.zeros((2, 40), device=dev)), lambda: dc.quantize_i8(f[:, 1:33])):
        with pytest.raises(dc.DcqError):
            call()


def test_example(dev):
    import importlib.util
    import os
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "moe_decode.py")
    spec = importlib.util.spec_from_file_location("moe_decode", path)
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    # int8 activations of 512 and 256 normal values: steps of about 3.2 sigma / 127, a third of one each way, so 0.8 % of a
    # value; through the norm's rows, two products, the gate and the second quantization the layer's own part is off by about 2 %
    assert all(v < 0.06 for v in example.main())


@pytest.mark.parametrize("m", [33, 48, 49, 61, 64])
@pytest.mark.parametrize("n,k", [(2304, 4080), (2304, 4096), (2681, 4112), (2688, 4096), (2690, 4096), (2704, 4096), (2561, 9728)])
def test_mul_mat_around_a_third_more_workgroups_than_cus(dev, m, n, k):
    """Two row tiles beside each other, both sides of what chooses them (N to 168 tiles of weight rows, a multiple of 8 of them,
    K from 4096 on): the sums, and the bits of one row by itself."""
    r = rng("a third more", m, n, k)
    w, ws = i8_rows(r, n, k)
    x, xs = i8_rows(r, m, k)
    res = r.standard_normal((m, n)).astype(np.float32)
    t = [gpu(a, dev) for a in (w, ws, x, xs, res)]
    y = dc.mul_mat_i8(*t[:4], r=t[4])
    check_product(y, w, ws, x, xs, res)
    for at in (0, 31, 32, m - 1):
        row = dc.mul_mat_i8(t[0], t[1], t[2][at:at + 1], t[3][at:at + 1], r=t[4][at:at + 1])
        assert torch.equal(row[0], y[at]), at


@pytest.mark.parametrize("m", [1, 12, 13, 100, 300, 700])
def test_a_dense_pair_is_one_expert(dev, m):
    """A dense layer's gate, up and down products by the experts' calls: one expert, one slot a token, weight 1. The down product's
    bits are mul_mat_i8's."""
    r = rng("one expert", m)
    n, k = 200, 528
    (wg, wgs), (wu, wus), (wd, wds) = i8_rows(r, n, k), i8_rows(r, n, k), i8_rows(r, k, n // 16 * 16)
    x, xs = i8_rows(r, m, k)
    h, hs = i8_rows(r, m, n // 16 * 16)
    res = r.standard_normal((m, k)).astype(np.float32)
    plan = dc.moe_plan(torch.zeros((m, 1), dtype=torch.int32, device=dev), 1)
    up = dc.moe_gate_up_i8(plan, gpu(wg, dev)[None], gpu(wgs, dev)[None], gpu(wu, dev)[None], gpu(wus, dev)[None], gpu(x, dev), gpu(xs, dev), 1)
    gate, lin = I.mul_mat(wg, wgs, x, xs), I.mul_mat(wu, wus, x, xs)
    ref = gate / (1 + np.exp(-gate)) * lin
    assert (np.abs(up.double().cpu().numpy() - ref) <= (12.1 + 3.01 * np.abs(gate)) * U * np.abs(ref) + 1e-36 * np.abs(lin)).all()
    t = [gpu(a, dev) for a in (wd, wds, h, hs)]
    y = dc.moe_down_i8(plan, t[0][None], t[1][None], t[2], t[3], torch.ones((m, 1), device=dev), r=gpu(res, dev))
    assert torch.equal(y, dc.mul_mat_i8(*t, r=gpu(res, dev)))
