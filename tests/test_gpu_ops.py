"""The operators on row tables and score rows (vectordb_amd.ops) against their definitions in 64 bits (oracle.ops_float64).

Tolerances count roundings.  u = 2^-24 is half a step of float32 relative to the value; a result of type t is rounded once
more, by at most eps(t) / 2 of its value or half its smallest step."""

import math

import numpy as np
import pytest
import torch

from oracle import ops_float64 as R

pytestmark = pytest.mark.gpu

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
U = R.UNIT


@pytest.fixture(scope="module")
def ops(native):
    from vectordb_amd import ops
    return ops


def rng_for(*what):
    return np.random.RandomState(sum(ord(c) * (i + 1) for i, c in enumerate(str(what))) % (2 ** 31))


def cuda(a, dtype=None):
    t = torch.as_tensor(np.ascontiguousarray(a)).cuda()
    return t if dtype is None else t.to(dtype)


def f64(t):
    return t.double().cpu().numpy()


def half_step(dtype, value):
    """largest error of one rounding of `value` to dtype"""
    info = torch.finfo(dtype)
    return np.maximum(np.abs(value) * (info.eps / 2), info.smallest_normal * info.eps / 2)


def check(got, want, tol, what=""):
    bad = ~(np.abs(got - want) <= tol) & ~((got == want) | (np.isnan(got) & np.isnan(want)))
    assert not bad.any(), (what, int(bad.sum()), np.argwhere(bad)[:3], got[bad][:3], want[bad][:3], np.broadcast_to(tol, got.shape)[bad][:3])


def padded(t, extra, shift):
    """The same matrix with a leading dimension `extra` longer, its first row `shift` elements behind an aligned address."""
    n, d = t.shape
    room = torch.full((n * (d + extra) + shift + 64,), 7.0, device="cuda", dtype=t.dtype)
    v = room[shift:shift + n * (d + extra)].view(n, d + extra)[:, :d]
    v.copy_(t)
    return v


# ---------------------------------------------------------------- lookup
@pytest.mark.parametrize("n", [1, 5, 700])
@pytest.mark.parametrize("dim", [1, 3, 8, 31, 128, 385, 2053])
@pytest.mark.parametrize("tin,tout", [("f32", "f32"), ("bf16", "bf16"), ("f16", "f16"), ("bf16", "f32"), ("f32", "bf16"), ("f16", "bf16")])
def test_lookup(ops, n, dim, tin, tout):
    rng = rng_for(n, dim, tin, tout)
    table = cuda(rng.randn(97, dim).astype(np.float32), TYPES[tin])
    rows = rng.randint(0, 97, n)
    rows[rng.rand(n) < 0.2] = -1
    for i, r in enumerate([96, 97, -(2 ** 63), 2 ** 63 - 1, 2 ** 32 + 3]):
        if i + 1 < n:
            rows[i + 1] = r
    got = ops.lookup(table, cuda(rows), scale=1.7, dtype=TYPES[tout])
    assert got.dtype == TYPES[tout] and tuple(got.shape) == (n, dim)
    want = R.lookup(f64(table), rows, float(np.float32(1.7)))
    # one product in float32, one rounding to the result's type
    check(f64(got), want, np.abs(want) * U + half_step(TYPES[tout], want * (1 + U)))
    assert torch.equal(got, ops.lookup(padded(table, 3, 1), cuda(rows), scale=1.7, dtype=TYPES[tout]))


def test_lookup_forms(ops, native):
    rng = rng_for("forms")
    x = rng.randn(500, 100).astype(np.float32)
    table, rows = cuda(x), cuda(rng.randint(-1, 500, (6, 10)))
    want = torch.where((rows >= 0)[..., None], table[rows.clamp_min(0)], 0.0)
    assert torch.equal(ops.lookup(table, rows), want)                      # the shape of a search's result
    out = torch.empty(6, 10, 100, device="cuda")
    assert ops.lookup(table, rows, out=out) is out and torch.equal(out, want)
    wide = torch.full((60, 130), 5.0, device="cuda")
    ops.lookup(table, rows.reshape(-1), out=wide[:, 7:107])
    assert torch.equal(wide[:, 7:107], want.reshape(60, 100)) and (wide[:, :7] == 5).all() and (wide[:, 107:] == 5).all()
    assert ops.lookup(table, rows[:0]).shape == (0, 10, 100)
    assert torch.equal(ops.lookup(table[:1].expand(500, 100), rows), torch.where((rows >= 0)[..., None], table[0], 0.0))
    assert torch.equal(ops.lookup(table[:0], rows), torch.zeros_like(want))
    # rows resident in a store, fp32 and bf16
    from vectordb_amd import _native
    for storage in ("f32", "bf16"):
        store = _native.RowStore(100, storage=storage)
        store.append(x)
        kept = table if storage == "f32" else table.bfloat16().float()
        assert torch.equal(ops.lookup(store, rows, scale=0.5), 0.5 * torch.where((rows >= 0)[..., None], kept[rows.clamp_min(0)], 0.0))
        store.truncate(300)                                                # numbers behind the end are unknown rows
        assert torch.equal(ops.lookup(store, rows), torch.where(((rows >= 0) & (rows < 300))[..., None], kept[rows.clamp(0, 299)], 0.0))
        store.close()


def test_lookup_far_offsets(ops):
    """Byte and element offsets beyond 32 bits."""
    table = torch.zeros((2 ** 31 + 2 ** 20) // 1024, 1024, device="cuda", dtype=torch.bfloat16)
    last = table.shape[0] - 1
    table[last] = 3.0
    table[last - 1000] = 2.0
    rows = torch.tensor([last, 0, last - 1000], device="cuda")
    assert torch.equal(ops.lookup(table, rows)[:, 5].float().cpu(), torch.tensor([3.0, 0.0, 2.0]))
    grad = torch.ones(3, 1024, device="cuda", dtype=torch.bfloat16)
    ops.lookup_grad(grad, rows, last + 1, out=table, accumulate=True)
    assert table[last, 1023].item() == 4.0 and table[last - 1000, 0].item() == 3.0 and table[0, 1].item() == 1.0
    assert table[1].abs().sum().item() == 0


# ---------------------------------------------------------------- gradient of a lookup
def grad_case(rng, kind, n, n_rows):
    if kind == "one":
        return np.full(n, n_rows // 2)
    if kind == "none":
        return np.full(n, -1)
    if kind == "all":
        return rng.permutation(max(n, n_rows))[:n] % n_rows
    r = np.minimum((n_rows ** rng.rand(n)).astype(np.int64) - 1 + rng.randint(0, 2, n), n_rows - 1)
    r[rng.rand(n) < 0.1] = rng.choice([-1, n_rows, 2 ** 40, -(2 ** 62)])
    return r


@pytest.mark.parametrize("kind", ["words", "one", "none", "all"])
@pytest.mark.parametrize("n,n_rows", [(0, 5), (1, 1), (31, 7), (32, 1), (33, 1000), (64, 64), (97, 3), (2048, 1500), (5000, 70000), (20000, 300)])
def test_lookup_grad(ops, kind, n, n_rows):
    rng = rng_for(kind, n, n_rows)
    dim = [1, 5, 16, 72, 130][(n + n_rows) % 5]
    rows = grad_case(rng, kind, n, n_rows).astype(np.int64)
    for tin, tout in (("f32", "f32"), ("bf16", "f32"), ("f16", "f16"), ("bf16", "bf16"))[(n % 2):]:
        g = cuda(rng.randn(n, dim).astype(np.float32), TYPES[tin])
        scale = float(np.float32(0.37))
        want, mag, cnt = R.lookup_grad(f64(g), rows, n_rows, scale)
        # cnt - 1 additions in float32, each off by u of a partial sum below `mag`, and the product with the scale
        tol = (cnt[:, None] + 1) * U * mag
        got = ops.lookup_grad(g, cuda(rows), n_rows, scale=0.37, dtype=TYPES[tout])
        check(f64(got), want, tol + half_step(TYPES[tout], np.abs(want) + tol), (tin, tout))
        assert torch.equal(got, ops.lookup_grad(padded(g, 5, 3) if n else g, cuda(rows), n_rows, scale=0.37, dtype=TYPES[tout]))
        # added to what is there; rows that nobody names keep their bits
        base = cuda(rng.randn(n_rows, dim).astype(np.float32), TYPES[tout])
        out = padded(base, 3, 1)
        ops.lookup_grad(g, cuda(rows), n_rows, scale=0.37, out=out, accumulate=True)
        total = f64(base) + want
        tol2 = tol + U * (np.abs(total) + tol)
        check(f64(out), total, tol2 + half_step(TYPES[tout], np.abs(total) + tol2), (tin, tout, "accumulate"))
        assert torch.equal(out[torch.from_numpy(cnt == 0).cuda()], base[torch.from_numpy(cnt == 0).cuda()])


def test_lookup_grad_many_rows(ops):
    """Three digits of the sort and more than a thousand blocks of it; sums of whole numbers are exact."""
    g = torch.Generator(device="cuda")
    g.manual_seed(5)
    n, n_rows = 2_500_000, 1_500_000
    rows = (n_rows ** torch.rand(n, device="cuda", generator=g).double()).long() - 1
    x = torch.randint(-3, 4, (n, 2), device="cuda", generator=g).float()
    got = ops.lookup_grad(x, rows, n_rows)
    want = torch.zeros(n_rows, 2, device="cuda", dtype=torch.float64).index_add_(0, rows, x.double())
    assert torch.equal(got.double(), want)


@pytest.mark.parametrize("n", [15, 16, 17, 1000, 4096, 4097, 8192, 8193, 12287, 12288, 12289])
@pytest.mark.parametrize("named", ["any", "two", "none", "one"])
def test_lookup_grad_sizes(ops, n, named):
    """Around the sizes at which the sort changes; rows named by nearly every position between rows that none names; rows that
    end inside a piece.  Sums of whole numbers are exact (below 2^24)."""
    rng = rng_for(n, named)
    for n_rows, dim, kind in ((7, 19, "f32"), (130, 13, "bf16"), (5000, 21, "f16"), (60000, 3, "bf16")):
        rows = {"any": rng.randint(-2, n_rows + 2, n), "two": rng.choice([3, 5], n), "none": np.full(n, -1), "one": np.full(n, n_rows - 1)}[named]
        x = rng.randint(-3, 4, (n, dim)).astype(np.float32)
        want = np.zeros((n_rows, dim))
        known = (rows >= 0) & (rows < n_rows)
        np.add.at(want, rows[known], x[known])
        got = ops.lookup_grad(cuda(x, TYPES[kind]), cuda(rows.astype(np.int64)), n_rows, dtype=torch.float32)
        assert (f64(got) == want).all()
        out = torch.full((n_rows, dim + 2), 7.0, device="cuda")
        ops.lookup_grad(cuda(x, TYPES[kind]), cuda(rows.astype(np.int64)), n_rows, out=out[:, :dim], accumulate=True)
        assert (f64(out[:, :dim]) == want + 7).all() and bool((out[:, dim:] == 7).all())


@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("n_rows,dim,n", [(1, 1, 0), (3, 1, 1), (5, 3, 1), (700, 33, 100), (100000, 7, 20), (90000, 5, 15000), (300, 129, 250)])
def test_lookup_grad_zeros(ops, kind, n_rows, dim, n):
    """Zeros over rows that lie back to back, at every offset from a 16-byte border, and over rows apart: all of them, nothing beside."""
    rng = rng_for("zeros", kind, n_rows)
    rows = rng.randint(0, n_rows, n)
    x = rng.randint(-3, 4, (n, dim)).astype(np.float32)
    want = np.zeros((n_rows, dim))
    np.add.at(want, rows, x)
    for off in range(9):
        room = torch.full((n_rows * dim + 20,), 7.0, device="cuda", dtype=TYPES[kind])
        out = room[off:off + n_rows * dim].view(n_rows, dim)
        ops.lookup_grad(cuda(x, TYPES[kind]), cuda(rows.astype(np.int64)), n_rows, out=out)
        assert (f64(out) == want).all() and bool((room[:off] == 7).all()) and bool((room[off + n_rows * dim:] == 7).all()), off
    room = torch.full((n_rows, dim + 3), 7.0, device="cuda", dtype=TYPES[kind])
    ops.lookup_grad(cuda(x, TYPES[kind]), cuda(rows.astype(np.int64)), n_rows, out=room[:, :dim])
    assert (f64(room[:, :dim]) == want).all() and bool((room[:, dim:] == 7).all())


@pytest.mark.parametrize("dim", [1, 2, 3, 4, 7, 8, 9, 255, 1023, 1024, 1025, 2047, 4099, 8193])
@pytest.mark.parametrize("tin,tout", [("f32", "f32"), ("bf16", "f32"), ("f16", "f16")])
def test_lookup_dimensions(ops, dim, tin, tout):
    """Rows of one piece to many, few rows and as many as change how a block takes them; nothing is written beside."""
    g = torch.Generator(device="cuda")
    g.manual_seed(dim)
    table = torch.randn(40, dim + 1, device="cuda", generator=g).to(TYPES[tin])[:, :dim]
    for n in (1, 9, 3000, 4_000_000 // dim):
        at = torch.randint(-1, 41, (n,), device="cuda", generator=g)
        room = torch.full((n, dim + 1), 7.0, device="cuda", dtype=TYPES[tout])
        ops.lookup(table, at, scale=0.5, out=room[:, :dim])
        want = (table.float()[at.clamp(0, 39)] * 0.5).to(TYPES[tout])
        want[(at < 0) | (at > 39)] = 0
        assert torch.equal(room[:, :dim], want) and bool((room[:, dim:] == 7).all()), n


@pytest.mark.parametrize("n", [1, 2, 63, 64, 65, 127, 128, 129])
@pytest.mark.parametrize("kind,tout", [("f32", "f32"), ("bf16", "f32"), ("f16", "f16")])
def test_lookup_grad_few(ops, n, kind, tout):
    """Few positions: rows of their own, one row for all, two that take turns, none; tables of one row to many."""
    rng = rng_for("few", n, kind)
    for n_rows, dim in ((1, 5), (70, 3), (500, 200), (300, 1030), (20, 4099), (3000, 390)):
        x = rng.randint(-3, 4, (n, dim)).astype(np.float32)
        grad = padded(cuda(x, TYPES[kind]), 3, 1)
        for rows in (rng.permutation(np.arange(n) % n_rows), np.full(n, n_rows - 1), np.arange(n) % 2, rng.randint(-2, n_rows + 2, n), np.full(n, -1)):
            want = np.zeros((n_rows, dim))
            known = (rows >= 0) & (rows < n_rows)
            np.add.at(want, rows[known], x[known])
            at = cuda(rows.astype(np.int64))
            room = torch.full((n_rows, dim + 1), 7.0, device="cuda", dtype=TYPES[tout])
            ops.lookup_grad(grad, at, n_rows, out=room[:, :dim])
            assert (f64(room[:, :dim]) == want).all() and bool((room[:, dim:] == 7).all()), (n_rows, dim)
            ops.lookup_grad(grad, at, n_rows, out=room[:, :dim], accumulate=True)
            assert (f64(room[:, :dim]) == 2 * want).all() and bool((room[:, dim:] == 7).all()), (n_rows, dim)


def test_lookup_grad_few_into_many(ops):
    """Few positions and a table whose zeros take longer than they do."""
    g = torch.Generator(device="cuda")
    g.manual_seed(4)
    for n, n_rows, dim in ((1, 90_000, 200), (20, 90_000, 200), (128, 17_000, 1000)):
        x = torch.randint(-3, 4, (n, dim), device="cuda", generator=g).float()
        at = torch.randint(-1, 9, (n,), device="cuda", generator=g) * (n_rows // 9)
        want = torch.zeros(n_rows, dim, device="cuda")
        want.index_add_(0, at[at >= 0], x[at >= 0])
        assert torch.equal(ops.lookup_grad(x, at, n_rows), want)
        assert torch.equal(ops.lookup_grad(x, at, n_rows, out=want.clone(), accumulate=True), 2 * want)


def test_lookup_grad_differences(ops):
    """The gradient of sum(w * lookup(table)) against the quotient of differences: linear, so the quotient is exact but for rounding."""
    rng = rng_for("differences")
    table, rows, w = rng.randn(20, 6), rng.randint(-1, 20, 40), rng.randn(40, 6).astype(np.float32)
    got = f64(ops.lookup_grad(cuda(w), cuda(rows), 20, scale=1.5))
    f = lambda t: float((w.astype(np.float64) * R.lookup(t, rows, 1.5)).sum())       # noqa: E731
    for r, c in ((0, 0), (7, 3), (19, 5), (4, 2)):
        up, down = table.copy(), table.copy()
        up[r, c] += 1e-3
        down[r, c] -= 1e-3
        assert abs((f(up) - f(down)) / 2e-3 - got[r, c]) < 1e-9 + 40 * U * 1.5 * np.abs(w).max() * 40


# ---------------------------------------------------------------- distillation
def distill_inputs(rng, n, vocab, k, dtype, ragged=True):
    z = cuda((2.5 * rng.randn(n, vocab)).astype(np.float32), dtype)
    t = np.sort(3 * rng.randn(n, k).astype(np.float32), axis=1)[:, ::-1].copy()
    at = rng.randint(0, vocab, (n, k)).astype(np.int64)
    if ragged and k > 0:
        for i in range(n):
            if i % 4 == 1:
                at[i, rng.randint(0, k):] = -1
            if i % 4 == 2:
                t[i, rng.randint(0, k)] = -np.inf
                at[i, rng.randint(0, k)] = vocab + rng.randint(0, 5)
        if n > 6:
            at[6] = -1
    return z, t, at


def distill_bounds(r, t, tau, vocab, k):
    """Error bounds of a row's loss, log-sum and gradient from the definition's own quantities.  An exponent (z - max) / tau
    has four roundings (difference, reciprocal of tau, log2(e) / tau, product), 2^x and exp are within 2 u; sums of m terms
    lose at most m u of the sum of magnitudes, m <= vocab / 256 + 16 in a thread and its joins, whose rescaling costs as
    much as an exponent again."""
    d, q, p = np.where(np.isfinite(r["d"]), -r["d"], 0.0), r["q"], r["p"]
    e_logs = U * (8 * float((q * d).sum()) + vocab / 256 + 16 + 8) + U * abs(r["logs"]) * 2 if np.isfinite(r["logs"]) else 0.0
    filled = p > 0
    dt = (np.max(t[filled]) - t[filled]) / tau if filled.any() else np.zeros(0)
    lp = np.abs(r["logp"][filled])
    e_lp = U * (4 * dt + 4 * lp + 4 * np.abs(t[filled]) / tau + k / 256 + 24)                    # of log p_j
    return e_logs, e_lp, filled


@pytest.mark.parametrize("vocab", [1, 2, 7, 255, 1000, 4097, 50021])
@pytest.mark.parametrize("k", [0, 1, 5, 64, 300])
@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
def test_distill(ops, vocab, k, kind):
    rng = rng_for(vocab, k, kind)
    dtype, n = TYPES[kind], 9 if vocab < 5000 else 3
    tau = [1.0, 0.7, 2.5][(vocab + k) % 3]
    z, t, at = distill_inputs(rng, n, vocab, k, dtype)
    lse = None
    if k % 2:
        lse = (np.max(np.where(np.isfinite(t), t, -9), axis=1) / tau + 0.3 + rng.rand(n)).astype(np.float32)
    w = rng.randn(n).astype(np.float32)
    w[0] = 0.0
    args = (cuda(t), cuda(at))
    kw = dict(temperature=tau, teacher_lse=None if lse is None else cuda(lse))
    loss, stats = ops.distill(z, *args, **kw)
    grad = ops.distill_grad(z, *args, stats, cuda(w), **kw)
    loss2, grad2 = ops.distill_step(z, *args, cuda(w), **kw)
    assert loss.shape == (n,) and stats.shape == (n, 2) and grad.dtype == dtype and grad.shape == (n, vocab)
    tau32 = float(np.float32(tau))
    for i in range(n):
        r = R.distill_row(f64(z[i]), t[i], at[i], tau32, None if lse is None else float(lse[i]))
        e_logs, e_lp, filled = distill_bounds(r, t[i].astype(np.float64), tau32, vocab, k)
        assert float(stats[i, 0]) == r["top"]
        assert abs(float(stats[i, 1]) - r["logs"]) <= e_logs
        p = r["p"][filled]
        gap = r["logp"][filled] - (r["d"][at[i][filled]] - r["logs"])
        e_gap = e_lp + e_logs + U * 4 * np.abs(r["d"][at[i][filled]])
        tol = tau32 ** 2 * float((p * (e_gap + np.abs(gap) * (e_lp + (k / 256 + 20) * U))).sum()) + 4 * U * abs(r["loss"])
        for got in (loss, loss2):
            assert abs(float(got[i]) - r["loss"]) <= tol, (i, float(got[i]), r["loss"], tol)
        want = w[i] * r["grad"]
        d = np.where(np.isfinite(r["d"]), -r["d"], 0.0)
        worst = float(e_lp.max()) if len(e_lp) else 0.0
        tol = np.abs(w[i]) * tau32 * (r["mass"] * r["q"] * (5 * U * d + e_logs + worst + (k / 256 + 24) * U) + r["target"] * (worst + (k + 8) * U))
        for got in (grad, grad2):
            check(f64(got[i]), want, tol + half_step(dtype, np.abs(want) + tol), i)
    # the same bits from rows that lie apart, and in place of the scores
    far = padded(z, 5, 3)
    assert torch.equal(ops.distill(far, *args, **kw)[0], loss)
    ops.distill_grad(far, *args, stats, cuda(w), out=far, **kw)
    assert torch.equal(far, grad)
    here = z.clone()
    loss3, _ = ops.distill_step(here, *args, cuda(w), out=here, **kw)
    assert torch.equal(here, grad2) and torch.equal(loss3, loss2)


@pytest.mark.parametrize("n,vocab,kind", [(2, 8190, "bf16"), (700, 4099, "f32"), (2, 16391, "f16"), (600, 9001, "bf16"), (3, 33001, "bf16"), (520, 32771, "f16"),
                                         (2, 65530, "f32"), (530, 65519, "bf16"), (1, 131057, "bf16"), (2, 131080, "f16"), (2, 300001, "bf16"), (1, 1000003, "f32")])
def test_distill_long_rows(ops, n, vocab, kind):
    """Rows around the sizes at which blocks change and rows are split, at every offset from a 16-byte border, both directions
    against sums in 64 bits on the GPU.  Bounds as in test_distill, for exponents up to 40."""
    g = torch.Generator(device="cuda")
    g.manual_seed(n * vocab)
    dtype, k = TYPES[kind], 11
    room = torch.randn(n * (vocab + 1) + 16, device="cuda", generator=g).mul_(2.5).to(dtype)
    z = room[3:3 + n * (vocab + 1)].view(n, vocab + 1)[:, :vocab]               # each row one element further from the border
    t = torch.randn(n, k, device="cuda", generator=g) * 3
    at = torch.randint(0, vocab, (n, k), device="cuda", generator=g)
    w = torch.rand(n, device="cuda", generator=g) + 0.5
    loss, stats = ops.distill(z, t, at)
    grad = ops.distill_grad(z, t, at, stats, w)
    loss2, grad2 = ops.distill_step(z, t, at, w)
    p = torch.softmax(t.double(), 1)
    logq = torch.log_softmax(z.double(), 1)
    want = (p * (p.log() - logq.gather(1, at))).sum(1)
    target = torch.zeros(n, vocab, device="cuda", dtype=torch.float64).scatter_add_(1, at, p)
    e_logs = U * (8 * 40 + vocab / 256 + 64)
    size = (p * (p.log() - logq.gather(1, at)).abs()).sum(1)
    for got in (loss, loss2):
        assert ((got.double() - want).abs() <= e_logs + U * 600 * size).all()
    assert torch.equal(stats[:, 0], z.float().amax(1))
    want = w.double()[:, None] * (logq.exp() - target)
    tol = w.double()[:, None] * (logq.exp() * (U * 300 + e_logs) + target * U * 300)
    half = torch.finfo(dtype).eps / 2
    for got in (grad, grad2):
        assert ((got.double() - want).abs() <= tol + torch.clamp(half * (want.abs() + tol), min=torch.finfo(dtype).smallest_normal * half)).all()
    outside = room.clone()
    assert torch.equal(ops.distill_step(z, t, at, w, out=z)[1], grad2)
    inside = outside[3:3 + n * (vocab + 1)].view(n, vocab + 1)
    inside[:, :vocab] = grad2
    assert torch.equal(room.float(), outside.float())                           # in place, and nothing beside the rows


@pytest.mark.parametrize("vocab", [1, 40, 900, 5000, 40_000])
def test_distill_long_lists(ops, vocab):
    """Lists of 1024 slots, longer than some rows: every place named many times, or one place by all."""
    rng = rng_for("long lists", vocab)
    n, k = 5, 1024
    z, t, at = distill_inputs(rng, n, vocab, k, torch.float32, ragged=False)
    at[1] = vocab - 1
    at[2, 100:] = -1
    at[3, ::2] = at[3, 1::2]
    w = rng.randn(n).astype(np.float32)
    loss, stats = ops.distill(z, cuda(t), cuda(at))
    grad = ops.distill_grad(z, cuda(t), cuda(at), stats, cuda(w))
    loss2, grad2 = ops.distill_step(z, cuda(t), cuda(at), cuda(w))
    for i in range(n):
        r = R.distill_row(f64(z[i]), t[i], at[i], 1.0)
        e_logs, e_lp, filled = distill_bounds(r, t[i].astype(np.float64), 1.0, vocab, k)
        # as in test_distill; up to k probabilities are added up one by one in a place
        worst = float(e_lp.max())
        for got in (loss, loss2):
            gap = np.abs(r["logp"][filled] - (r["d"][at[i][filled]] - r["logs"]))
            tol = float((r["p"][filled] * (worst + e_logs + U * 200 + gap * (worst + 40 * U))).sum()) + 4 * U * abs(r["loss"])
            assert abs(float(got[i]) - r["loss"]) <= tol, (i, float(got[i]), r["loss"], tol)
        d = np.where(np.isfinite(r["d"]), -r["d"], 0.0)
        tol = np.abs(w[i]) * (r["mass"] * r["q"] * (5 * U * d + e_logs + worst + (k / 64 + 24) * U) + r["target"] * (worst + (k + 8) * U))
        for got in (grad, grad2):
            check(f64(got[i]), w[i] * r["grad"], tol + half_step(torch.float32, np.abs(w[i] * r["grad"]) + tol), i)


def test_distill_many_rows(ops):
    """More rows than one launch takes: the last ones are what they are by themselves."""
    n, vocab, k = (1 << 21) + 7, 9, 3
    g = torch.Generator(device="cuda")
    g.manual_seed(1)
    z, t = torch.randn(n, vocab, device="cuda", generator=g).bfloat16(), torch.randn(n, k, device="cuda", generator=g)
    at, w = torch.randint(0, vocab, (n, k), device="cuda", generator=g), torch.rand(n, device="cuda", generator=g)
    loss, stats = ops.distill(z, t, at)
    grad = ops.distill_grad(z, t, at, stats, w)
    loss2, grad2 = ops.distill_step(z, t, at, w)
    for lo, hi in ((0, 20), (n - 20, n)):
        part = z[lo:hi], t[lo:hi], at[lo:hi]
        one, its = ops.distill(*part)
        assert torch.equal(loss[lo:hi], one) and torch.equal(stats[lo:hi], its)
        assert torch.equal(grad[lo:hi], ops.distill_grad(*part, its, w[lo:hi]))
        one, its = ops.distill_step(*part, w[lo:hi])
        assert torch.equal(loss2[lo:hi], one) and torch.equal(grad2[lo:hi], its)


def test_sample_many_rows(ops):
    n, vocab = (1 << 21) + 7, 9
    g = torch.Generator(device="cuda")
    g.manual_seed(1)
    z, u = torch.randn(n, vocab, device="cuda", generator=g), torch.rand(n, device="cuda", generator=g)
    top_p = torch.rand(n, device="cuda", generator=g)
    row, logp = ops.sample(z, u, top_p=top_p)
    for lo, hi in ((0, 20), (n - 20, n)):
        one, its = ops.sample(z[lo:hi], u[lo:hi], top_p=top_p[lo:hi])
        assert torch.equal(row[lo:hi], one) and torch.equal(logp[lo:hi], its)


def test_lookup_many_rows(ops):
    n, dim = (1 << 23) + 5, 1030
    table = torch.randn(100, dim, device="cuda")
    at = torch.arange(n, device="cuda") % 101                                   # 100: no row
    out = ops.lookup(table, at, dtype=torch.bfloat16)
    for lo, hi in ((0, 300), (n - 300, n)):
        assert torch.equal(out[lo:hi], ops.lookup(table, at[lo:hi], dtype=torch.bfloat16))
    assert torch.equal(out[n - 1], table[(n - 1) % 101].bfloat16())


def test_distill_differences(ops):
    rng = rng_for("distill differences")
    z, t, at = distill_inputs(rng, 8, 40, 6, torch.float32)
    loss, stats = ops.distill(z, cuda(t), cuda(at), temperature=1.3)
    grad = f64(ops.distill_grad(z, cuda(t), cuda(at), stats, torch.ones(8, device="cuda"), temperature=1.3))
    z64, h = f64(z), 1e-4
    for i in range(8):
        for v in range(0, 40, 7):
            up, down = z64[i].copy(), z64[i].copy()
            up[v] += h
            down[v] -= h
            q = (R.distill_row(up, t[i], at[i], 1.3)["loss"] - R.distill_row(down, t[i], at[i], 1.3)["loss"]) / (2 * h)
            # third derivatives of the loss are below 1 / tau: the quotient is off by h^2 / 6 at most; float32 gradients by 1e-6
            assert abs(q - grad[i, v]) < 1e-8 + 2e-6, (i, v, q, grad[i, v])


@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
def test_distill_odd_rows(ops, kind):
    """Masked scores, rows without anything, NaN and infinities that stay in their row, slots that share a place."""
    dtype = TYPES[kind]
    low = torch.finfo(dtype).min
    vocab, inf = 700, math.inf
    rng = rng_for("odd", kind)
    z = cuda(rng.randn(10, vocab).astype(np.float32), dtype)
    t = np.zeros((10, 4), np.float32) + np.array([2.0, 1.0, 0.5, 0.0], np.float32)
    at = np.tile(np.array([3, 10, 500, 699], np.int64), (10, 1))
    z[0, 20:] = -inf; at[0] = [0, 1, 2, 3]                 # most of the row masked
    z[1, 20:] = low; at[1] = [0, 1, 2, 3]                  # the same with the type's lowest value
    z[2, :] = low                                          # every score the lowest: uniform
    z[3, :] = -inf                                         # nothing left: loss +inf, q = 0
    z[4, 10] = -inf                                        # the teacher names a masked place: loss +inf
    z[5, 7] = math.nan
    z[6, 7] = math.nan; at[6] = -1                         # nothing filled: loss 0, gradient 0
    t[7] = -inf                                            # the same by scores
    at[8] = [5, 5, 5, 5]                                   # one place four times
    z[9, 50] = inf
    w = torch.ones(10, device="cuda")
    for tau in (1.0, 0.5):
        loss, stats = ops.distill(z, cuda(t), cuda(at), temperature=tau)
        grad = ops.distill_grad(z, cuda(t), cuda(at), stats, w, temperature=tau)
        loss2, grad2 = ops.distill_step(z, cuda(t), cuda(at), w, temperature=tau)
        for ls, gr in ((loss, grad), (loss2, grad2)):
            l, g = f64(ls), f64(gr)
            for i in (0, 1, 2, 8):
                r = R.distill_row(f64(z[i]), t[i], at[i], tau)
                # few terms of moderate size: 100 roundings cover the row
                assert abs(l[i] - r["loss"]) <= 100 * U * max(1, abs(r["loss"])), (i, l[i], r["loss"])
                tol = 100 * U * (r["q"] + r["target"])
                check(g[i], r["grad"], tol + half_step(dtype, np.abs(r["grad"]) + tol), i)
            assert l[3] == inf and l[4] == inf and np.isnan(l[5]) and l[6] == 0 and l[7] == 0 and np.isnan(l[9])
            p = R.teacher_probabilities(t[3].astype(np.float64), at[3], vocab, tau)[0]
            want = np.zeros(vocab)
            want[at[3]] = -tau * p
            check(g[3], want, 100 * U + half_step(dtype, want))
            assert np.isfinite(g[4]).all() and g[4][10] < 0 and np.isnan(g[5]).all() and np.isnan(g[9]).all()
            assert (g[6] == 0).all() and (g[7] == 0).all()
        assert (f64(ops.distill_grad(z, cuda(t), cuda(at), stats, 0 * w, temperature=tau)) == 0).all()
        assert (f64(ops.distill_step(z, cuda(t), cuda(at), 0 * w, temperature=tau)[1]) == 0).all()


def test_distill_shapes(ops):
    z = torch.randn(6, 50, device="cuda")
    t, at = torch.randn(6, 4, device="cuda"), torch.randint(0, 50, (6, 4), device="cuda")
    want = ops.distill(z, t, at)[0]
    assert torch.equal(ops.distill(z, torch.cat([t, t], 1)[:, :4], torch.cat([at, at, at], 1)[:, 4:8])[0], want)     # lists that lie apart
    one = ops.distill(z, t[:1].expand(6, 4), at[:1].expand(6, 4))[0]                                               # one list for all
    assert torch.equal(one, ops.distill(z, t[:1].repeat(6, 1), at[:1].repeat(6, 1))[0])
    shared = ops.distill(z[:1].expand(6, 50), t, at)[0]                                                             # one score row for all
    assert torch.equal(shared, ops.distill(z[:1].repeat(6, 1), t, at)[0])
    assert ops.distill(z[:0], t[:0], at[:0])[0].shape == (0,)
    assert ops.distill_step(z[:0], t[:0], at[:0], torch.zeros(0, device="cuda"))[1].shape == (0, 50)


# ---------------------------------------------------------------- sampling
def sample_oracle(z, u, **kw):
    n = len(z)
    per = lambda v, i: v[i] if isinstance(v, np.ndarray) else v       # noqa: E731
    got = [R.sample_row(z[i], float(u[i]), **{k: (per(v, i) if k != "allowed" else (v if v is None or v.ndim == 1 else v[i])) for k, v in kw.items()})
           for i in range(n)]
    return np.array([g[0] for g in got]), np.array([g[1] for g in got])


def words_of(allowed):
    from vectordb_amd import _native
    rows = np.atleast_2d(allowed)
    w = np.stack([_native.pack_mask(r) for r in rows]).view(np.int32)
    return cuda(w if allowed.ndim == 2 else w[0])


def sample_check(ops, z, u, allowed=None, distances=False, **kw):
    scores = f64(z)
    rows, logp = ops.sample(z, cuda(u), mask_words=None if allowed is None else words_of(allowed), distances=distances,
                            **{k: (cuda(v) if isinstance(v, np.ndarray) else v) for k, v in kw.items()})
    okw = {"tau": kw.get("temperature", 1.0), "top_k": kw.get("top_k", 0), "top_p": kw.get("top_p", 1.0), "min_p": kw.get("min_p", 0.0), "allowed": allowed}
    okw = {k: (0 if v is None and k == "top_k" else float(np.float32(v)) if isinstance(v, float) else
               v.astype(np.float64) if isinstance(v, np.ndarray) and v.dtype == np.float32 else v) for k, v in okw.items()}
    want, wlog = sample_oracle(-scores if distances else scores, u, **okw)
    got = rows.cpu().numpy()
    assert np.array_equal(got, want), (np.flatnonzero(got != want)[:5], got[got != want][:5], want[got != want][:5], kw)
    # a quotient and a logarithm in 64 bits, rounded to float32
    check(f64(logp), wlog, U * np.abs(wlog) + 1e-10)
    return got


@pytest.mark.parametrize("vocab", [1, 2, 31, 64, 1000, 8191, 32768, 50021])
@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("masked", [False, True])
def test_sample_settings(ops, vocab, kind, masked):
    rng = rng_for("sample", vocab, kind, masked)
    n = 24
    z = cuda((2.5 * rng.randn(n, vocab)).astype(np.float32), TYPES[kind])
    u = rng.rand(n).astype(np.float32)
    u[:3] = [0.0, 1 - 2.0 ** -24, 0.5]
    allowed = rng.rand(n, vocab) < np.linspace(0, 1, n)[:, None] if masked else None       # row 0: nothing, row n - 1: everything
    choose = lambda *v: rng.choice(v, n)                                                  # noqa: E731
    sample_check(ops, z, u, allowed)
    sample_check(ops, z, u, allowed, temperature=0.0)
    sample_check(ops, z, u, allowed, temperature=0.8, top_k=7)
    sample_check(ops, z, u, allowed, temperature=1.3, top_p=0.9)
    sample_check(ops, z, u, allowed, min_p=0.1)
    sample_check(ops, z, u, allowed, temperature=choose(0.0, 0.3, 1.0, 4.0).astype(np.float32), top_k=choose(0, 1, 3, 50, 2000, vocab, vocab + 1).astype(np.int32),
                 top_p=choose(0.0, 0.1, 0.5, 0.95, 0.999, 1.0).astype(np.float32), min_p=choose(0.0, 0.001, 0.2, 1.0, 3.0).astype(np.float32))


@pytest.mark.parametrize("top_k,top_p,min_p", [(0, 1.0, 0.0), (5, 1.0, 0.0), (700, 1.0, 0.0), (0, 0.25, 0.0), (0, 0.7, 0.0), (300, 0.5, 0.0), (9, 0.34, 1.0), (1, 0.0, 0.5)])
def test_sample_ties(ops, top_k, top_p, min_p):
    """Rows of few distinct values: every border falls among equal scores, which rank by row number."""
    rng = rng_for("ties", top_k, top_p)
    n, vocab = 40, 1537
    z = rng.randint(-2, 3, (n, vocab)).astype(np.float32)
    z[:8] = 1.0                                       # all equal
    z[8:12] = -0.0
    z[8:12, ::3] = 0.0                                # -0 and +0 are one value
    u = rng.rand(n).astype(np.float32)
    u[:6] = [0.0, 0.25, 0.5, 0.75, 1 - 2.0 ** -24, 1 / 3]
    allowed = rng.rand(vocab) < 0.7
    for kind in ("f32", "bf16"):
        sample_check(ops, cuda(z, TYPES[kind]), u, top_k=top_k, top_p=top_p, min_p=min_p)
        sample_check(ops, cuda(z, TYPES[kind]), u, allowed, top_k=top_k, top_p=top_p, min_p=min_p, temperature=0.5)


@pytest.mark.parametrize("top_k,top_p,min_p", [(0, 1.0, 0.0), (5, 1.0, 0.0), (2500, 0.9, 0.0), (30000, 1.0, 0.0), (0, 0.25, 0.0), (0, 0.7, 0.0), (0, 1.0, 0.4), (0, 0.95, 0.9)])
def test_sample_ties_long(ops, top_k, top_p, min_p):
    """The same in rows that the whole chip goes through: thousands of equal scores at a border, rows of one value, filters
    that leave single scores, whole stretches or nothing."""
    rng = rng_for("ties long", top_k, top_p)
    n, vocab = 12, 40_009
    z = rng.randint(-2, 3, (n, vocab)).astype(np.float32)
    z[:3] = 1.0
    z[3] = -0.0
    z[3, ::3] = 0.0
    z[4, 20_000:] = np.finfo(np.float32).min
    z[5] = -np.inf
    z[5, [7, 40_008]] = 0.0
    z[6, ::2] = math.nan
    u = rng.rand(n).astype(np.float32)
    u[:3] = [0.0, 0.5, 1 - 2.0 ** -24]
    allowed = rng.rand(n, vocab) < 0.7
    allowed[7] = False
    allowed[8] = False
    allowed[8, 33_333] = True
    allowed[9, :39_000] = False
    for kind in ("f32", "f16"):
        with np.errstate(over="ignore"):
            scores = cuda(z, TYPES[kind])
        sample_check(ops, scores, u, top_k=top_k, top_p=top_p, min_p=min_p)
        sample_check(ops, scores, u, allowed, top_k=top_k, top_p=top_p, min_p=min_p, temperature=0.5)
    sample_check(ops, cuda(-z), u, allowed[10], distances=True, top_k=top_k, top_p=top_p, min_p=min_p)


def test_sample_long_batches(ops):
    """More long rows than are worked on at a time, each with settings and a filter of its own: what they are by themselves."""
    g = torch.Generator(device="cuda")
    g.manual_seed(8)
    n, vocab = 2050, 33_000
    r = lambda *s: torch.rand(*s, device="cuda", generator=g)               # noqa: E731
    z, u = torch.randn(n, vocab, device="cuda", generator=g).bfloat16() * 2, r(n)
    tau, top_p, min_p = r(n) * 2, r(n) * 1.2, (r(n) - 0.5).clamp(min=0)
    top_k = torch.randint(0, 4, (n,), device="cuda", generator=g, dtype=torch.int32) * 60
    words = torch.randint(-2 ** 31, 2 ** 31, (n, (vocab + 31) // 32), device="cuda", generator=g).int()
    row, logp = ops.sample(z, u, tau, top_k, top_p, min_p, words)
    for i in (0, 1, 1023, 1024, 1025, 2047, 2048, 2049):
        s = slice(i, i + 1)
        one = ops.sample(z[s], u[s], tau[s], top_k[s], top_p[s], min_p[s], words[s])
        assert torch.equal(row[s], one[0]) and torch.equal(logp[s], one[1]), i
        bits = words[i].cpu().numpy().view(np.uint32)
        allowed = np.unpackbits(bits.view(np.uint8), bitorder="little")[:vocab].astype(bool)
        want, wlog = R.sample_row(f64(z[i]), float(u[i]), float(tau[i]), int(top_k[i]), float(top_p[i]), float(min_p[i]), allowed)
        assert int(row[i]) == want and abs(float(logp[i]) - wlog) <= U * abs(wlog) + 1e-10, i


def test_sample_odd_rows(ops):
    rng = rng_for("odd sample")
    inf = math.inf
    z = rng.randn(12, 300).astype(np.float32)
    z[0] = -inf
    z[1] = math.nan
    z[2, ::2] = math.nan
    z[3, :299] = -inf
    z[4, [5, 9]] = inf
    z[5] = np.finfo(np.float32).min
    z[6, 10:] = np.finfo(np.float32).min
    z[7] = 100 * z[7]
    z[8, 0] = 1e30
    allowed = np.ones((12, 300), bool)
    allowed[9] = False
    allowed[10, :] = False
    allowed[10, 299] = True
    z[11, 7] = math.nan
    allowed[11, 7] = False
    u = rng.rand(12).astype(np.float32)
    for kw in ({}, {"top_p": 0.9}, {"top_k": 3}, {"min_p": 0.3}, {"temperature": 0.0}, {"temperature": 1e30}, {"temperature": 1e-30, "top_k": 9, "top_p": 0.5}):
        for kind in ("f32", "bf16"):
            got = sample_check(ops, cuda(z, TYPES[kind]), u, allowed, **kw)
            assert got[0] == -1 and got[1] == -1 and got[3] == 299 and got[9] == -1 and got[10] == 299
    assert ops.sample(torch.zeros(0, 5, device="cuda"), torch.zeros(0, device="cuda"))[0].shape == (0,)


def test_sample_forms(ops):
    rng = rng_for("sample forms")
    z = rng.randn(16, 900).astype(np.float32)
    u = rng.rand(16).astype(np.float32)
    want = sample_check(ops, cuda(z), u, top_k=40)
    assert np.array_equal(sample_check(ops, cuda(-z), u, distances=True, top_k=40), want)
    assert np.array_equal(ops.sample(padded(cuda(z), 7, 3), cuda(u), top_k=40)[0].cpu().numpy(), want)
    allowed = rng.rand(900) < 0.3
    shared = sample_check(ops, cuda(z), u, allowed, top_p=0.8)
    w = words_of(allowed)
    assert np.array_equal(ops.sample(cuda(z), cuda(u), top_p=0.8, mask_words=w[None].expand(16, -1))[0].cpu().numpy(), shared)
    assert np.array_equal(ops.sample(cuda(z), cuda(u), top_p=0.8, mask_words=w.view(torch.uint32))[0].cpu().numpy(), shared)


def test_sample_frequencies(ops):
    """Evenly spaced uniform numbers visit each row as often as its probability says, to one number."""
    n = 4096
    z = torch.tensor([[0.0, 1.0, -1.0, 2.0, 0.5]], device="cuda").expand(n, 5)
    u = (torch.arange(n, device="cuda") + 0.5) / n
    got = torch.bincount(ops.sample(z, u.float())[0], minlength=5).cpu().numpy()
    p = np.exp([0.0, 1.0, -1.0, 2.0, 0.5])
    assert (np.abs(got - n * p / p.sum()) <= 1).all()


def test_sample_large(ops):
    """A million scores a row, a row of them all equal, and the repeat of the same bits."""
    g = torch.Generator(device="cuda")
    g.manual_seed(3)
    z = 2.0 * torch.randn(3, 1_000_003, device="cuda", generator=g)
    z[1] = 0.25
    u = np.array([0.3, 0.7, 0.9], np.float32)
    for kw in ({}, {"top_k": 5000}, {"top_p": 0.99}, {"min_p": 0.02}):
        sample_check(ops, z, u, **kw)


# ---------------------------------------------------------------- refusals
def test_refusals(ops):
    f, i, u = torch.zeros(4, 8, device="cuda"), torch.zeros(4, dtype=torch.int64, device="cuda"), torch.zeros(4, device="cuda")
    lists = (torch.zeros(4, 2, device="cuda"), torch.zeros(4, 2, dtype=torch.int64, device="cuda"))
    stats = torch.zeros(4, 2, device="cuda")
    for text, call in [
        ("float32, bfloat16 or float16", lambda: ops.lookup(f.double(), i)), ("two dimensions", lambda: ops.lookup(f[0], i)),
        ("int64", lambda: ops.lookup(f, i.int())), ("contiguous", lambda: ops.lookup(f.t(), i)), ("contiguous", lambda: ops.lookup(f, i[::2])),
        ("shape", lambda: ops.lookup(f, i, out=f[:2])), ("apart", lambda: ops.lookup(f, i, out=f[:1].expand(4, 8))),
        ("dtype", lambda: ops.lookup(f, i, dtype=torch.int32)), ("GPU", lambda: ops.lookup(f, i.cpu())),
        ("shape", lambda: ops.lookup_grad(f[:3], i, 5)), ("out", lambda: ops.lookup_grad(f, i, 5, accumulate=True)),
        ("shape", lambda: ops.lookup_grad(f, i, 5, out=f)), ("bad sizes", lambda: ops.lookup_grad(f, i, -1)),
        ("shape", lambda: ops.distill(f, lists[0][:3], lists[1])), ("float32", lambda: ops.distill(f, lists[0].half(), lists[1])),
        ("int64", lambda: ops.distill(f, lists[0], lists[1].int())), ("temperature", lambda: ops.distill(f, *lists, temperature=0.0)),
        ("teacher_lse", lambda: ops.distill(f, *lists, teacher_lse=u[:3])), ("slots", lambda: ops.distill(f, torch.zeros(4, 1025, device="cuda"),
                                                                                                      torch.zeros(4, 1025, device="cuda").long())),
        ("stats", lambda: ops.distill_grad(f, *lists, stats[:3], u)), ("grad_loss", lambda: ops.distill_grad(f, *lists, stats, u.double())),
        ("shape", lambda: ops.distill_step(f, *lists, u, out=f[:3])), ("at least one", lambda: ops.distill(f[:, :0], *lists)),
        ("uniforms", lambda: ops.sample(f, u[:3])), ("top_k", lambda: ops.sample(f, u, top_k=1.5)), ("top_k", lambda: ops.sample(f, u, top_k=i)),
        ("temperature", lambda: ops.sample(f, u, temperature=torch.zeros(3, device="cuda"))), ("filter", lambda: ops.sample(f, u, mask_words=u)),
        ("filter", lambda: ops.sample(f, u, mask_words=torch.zeros(3, 1, dtype=torch.int32, device="cuda"))),
        ("at least one", lambda: ops.sample(f[:, :0], u)),
    ]:
        with pytest.raises(ValueError, match=text):
            call()


# ---------------------------------------------------------------- workspaces
def test_workspaces_are_kept_to(ops, monkeypatch):
    """No call writes before or behind the bytes that its workspace function names, and none reads what was there before."""
    guards = []

    def workspace(fn, *sizes):
        need = ops._workspace_bytes(fn, *sizes)
        t = torch.randint(0, 256, (need + 1024,), device="cuda", dtype=torch.uint8)
        guards.append((t, t.clone(), need, fn, sizes))
        return t, t.data_ptr() + 512, need

    def run(call):
        guards.clear()
        monkeypatch.setattr(ops, "_workspace", workspace)
        got = call()
        monkeypatch.undo()
        want = call()
        for t, before, need, fn, sizes in guards:
            assert torch.equal(t[:512], before[:512]) and torch.equal(t[512 + need:], before[512 + need:]), (fn, sizes)
        for x, y in zip(got, want):
            assert torch.equal(x, y), guards[0][3:]

    g = torch.Generator(device="cuda")
    g.manual_seed(2)
    r = lambda *s: torch.randn(*s, device="cuda", generator=g)               # noqa: E731
    for n, n_rows, dim in ((1, 5, 3), (33, 7, 9), (100, 1000, 5), (4097, 90, 33), (12288, 60, 16), (12289, 60, 16), (20000, 300000, 6), (70000, 5000, 130)):
        x, at = r(n, dim), torch.randint(-1, n_rows, (n,), device="cuda", generator=g)
        run(lambda: (ops.lookup_grad(x, at, n_rows),))
    for dtype in (torch.float32, torch.bfloat16):
        for n, vocab in ((1, 10), (5, 32768), (3, 65527), (3, 65528), (2, 65537), (1, 131072), (130, 70001), (600, 65536), (600, 65540), (1, 1000003)):
            z, t, at, w = r(n, vocab).to(dtype), r(n, 4), torch.randint(-1, vocab, (n, 4), device="cuda", generator=g), r(n)
            run(lambda: ops.distill(z, t, at))
            run(lambda: ops.distill_step(z, t, at, w))
        for n, vocab in ((3, 32768), (3, 32769), (2, 40_000), (17, 131072), (2, 600_001)):
            z, u = r(n, vocab).to(dtype) * 2, torch.rand(n, device="cuda", generator=g)
            for kw in ({}, {"top_k": 90}, {"top_p": 0.9}, {"min_p": 0.001}):
                run(lambda: ops.sample(z, u, **kw))


# ---------------------------------------------------------------- together
def together(ops, table, tokens, queries, teacher, at, weight, uniforms):
    """A training step of the rows and an answer: look rows up, score them, distill, send the gradient back to the rows; draw from the scores."""
    x = ops.lookup(table, tokens, scale=0.5)
    scores = x @ queries.t()
    loss, d_scores = ops.distill_step(scores, teacher, at, weight, temperature=2.0)
    d_table = ops.lookup_grad(d_scores @ queries, tokens, table.shape[0], scale=0.5)
    drawn, logp = ops.sample(scores, uniforms, temperature=0.7, top_k=20, top_p=0.9)
    answer = ops.lookup(queries, drawn)
    return loss, d_table, drawn, logp, answer


def together_inputs(seed, n=64, n_rows=300, dim=32, vocab=500):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    r = lambda *s: torch.randn(s, device="cuda", generator=g)         # noqa: E731
    tokens = torch.randint(-1, n_rows, (n,), device="cuda", generator=g)
    at = torch.randint(0, vocab, (n, 8), device="cuda", generator=g)
    at[::9] = -1
    return r(n_rows, dim), tokens, r(vocab, dim), r(n, 8), at, torch.rand(n, device="cuda", generator=g), torch.rand(n, device="cuda", generator=g)


def test_together(ops):
    """The chain's gradient against differences of the whole chain in 64 bits, and its draws against the definition."""
    table, tokens, queries, teacher, at, weight, uniforms = inputs = together_inputs(1)
    loss, d_table, drawn, logp, answer = together(ops, *inputs)
    T, tok, Q = f64(table), tokens.cpu().numpy(), f64(queries)
    t64, a64, w64 = f64(teacher), at.cpu().numpy(), f64(weight)

    def objective(tab):
        s = R.lookup(tab, tok, 0.5) @ Q.T
        return sum(w64[i] * R.distill_row(s[i], t64[i], a64[i], 2.0)["loss"] for i in range(len(tok)))

    got = f64(d_table)
    for r, c in ((int(tok[1]) if tok[1] >= 0 else 0, 0), (int(tok[2]), 5), (17, 31)):
        up, down = T.copy(), T.copy()
        up[r, c] += 1e-4
        down[r, c] -= 1e-4
        q = (objective(up) - objective(down)) / 2e-4
        # sums of 500 products of size 1 in float32, scores up to 20: about 1e-4 of the value is far above 1000 u
        assert abs(q - got[r, c]) <= 1e-4 * max(1.0, abs(got).max()), (r, c, q, got[r, c])
    scores = f64(ops.lookup(table, tokens, scale=0.5) @ queries.t())
    want, _ = sample_oracle(scores, f64(uniforms), tau=float(np.float32(0.7)), top_k=20, top_p=float(np.float32(0.9)), min_p=0.0, allowed=None)
    assert np.array_equal(drawn.cpu().numpy(), want)
    assert torch.equal(answer, queries[drawn])


def test_captured_and_replayed(ops):
    """Two graphs of the chain, replayed in turn with new inputs and eager work between, against eager results."""
    graphs = []
    for seed in (11, 12):
        inputs = [t.clone() for t in together_inputs(seed)]
        side = torch.cuda.Stream()
        with torch.cuda.stream(side):
            together(ops, *inputs)
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs = together(ops, *inputs)
        graphs.append((g, inputs, outs))
    for turn in range(3):
        for k, (g, inputs, outs) in enumerate(graphs):
            for t, new in zip(inputs, together_inputs(100 + 10 * turn + k)):
                t.copy_(new)
            g.replay()
            want = together(ops, *inputs)
            torch.cuda.synchronize()
            for a, b in zip(outs, want):
                assert torch.equal(a, b), (turn, k)


def test_captured_large(ops):
    """Calls of several launches, captured together and replayed with new inputs and eager work between, against eager results."""
    def inputs(seed):
        g = torch.Generator(device="cuda")
        g.manual_seed(seed)
        r = lambda *s: torch.randn(*s, device="cuda", generator=g)           # noqa: E731
        return (r(20000, 24), torch.randint(-1, 9000, (20000,), device="cuda", generator=g), r(3, 140_001) * 2, r(3, 6),
                torch.randint(-1, 140_001, (3, 6), device="cuda", generator=g), torch.rand(3, device="cuda", generator=g))

    def calls(x, at, z, t, rows, u):
        return (ops.lookup_grad(x, at, 9000), ops.lookup_grad(x[:3000], at[:3000], 9000), *ops.distill(z, t, rows), *ops.distill_step(z, t, rows, u),
                *ops.sample(z, u, top_p=0.9), *ops.sample(z[:, :20_000], u, top_p=0.8), *ops.sample(z, u, top_k=300))

    ins = [t.clone() for t in inputs(1)]
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        calls(*ins)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        outs = calls(*ins)
    for turn in range(4):
        for t, new in zip(ins, inputs(50 + turn)):
            t.copy_(new)
        g.replay()
        want = calls(*ins)
        torch.cuda.synchronize()
        for k, (a, b) in enumerate(zip(outs, want)):
            assert torch.equal(a, b), (turn, k)


def test_two_streams(ops):
    """Calls on two streams at once, each with a workspace of its own."""
    ins = [together_inputs(s, n=512, n_rows=900) for s in (21, 22)]
    want = [together(ops, *i) for i in ins]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(4):
        got = []
        for s, i in zip(streams, ins):
            with torch.cuda.stream(s):
                got.append(together(ops, *i))
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert all(torch.equal(x, y) for x, y in zip(a, b))
