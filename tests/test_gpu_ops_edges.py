"""The operators on row tables and score rows at places that random inputs hardly reach, against their definitions in 64
bits (oracle.ops_float64).  Tolerances as in test_gpu_ops."""

import numpy as np
import pytest
import torch

from oracle import ops_float64 as R
from test_gpu_ops import TYPES, U, cuda, f64, ops, rng_for, sample_check  # noqa: F401 (ops is a fixture)

pytestmark = pytest.mark.gpu


# ---------------------------------------------------------------- sampling: rows at the beginning, lists beyond all pairs
def uniforms_for(z, rows, kept):
    """Uniform numbers in the middle of the shares that `rows` have among the rows `kept` of the scores z (temperature 1)."""
    w = np.where(kept, np.exp(z - z.max()), 0.0)
    reach = np.cumsum(w)
    return ((reach[rows] - 0.5 * w[rows]) / reach[-1]).astype(np.float32)


@pytest.mark.parametrize("vocab", [4097, 5002, 30522, 50257, 100277])
@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_sample_draws_of_the_first_rows(ops, vocab, kind):  # noqa: F811
    """Each of the first 64 rows drawn out of lists of 300 to 1500."""
    rng = rng_for("first rows", vocab, kind)
    z = -12 + rng.rand(vocab)
    z[rng.permutation(np.arange(64, vocab))[:1400]] = 2 * rng.rand(1400)
    z[:64] = 2.2 + 0.5 * rng.rand(64)                      # the best: they remain whatever the setting
    scores = cuda(z[None].astype(np.float32), TYPES[kind])
    z = f64(scores)[0]
    order = np.argsort(-z, kind="stable")
    rows = np.arange(64)
    for kw, keep in (({"top_k": 300}, 300), ({"top_k": 1000}, 1000), ({"min_p": 0.03}, 1464)):
        kept = np.zeros(vocab, bool)
        kept[order[:keep]] = True
        got = sample_check(ops, scores.expand(64, vocab), uniforms_for(z, rows, kept), **kw)
        assert np.array_equal(got, rows)


@pytest.mark.parametrize("vocab", [4097, 30522, 50257])
@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_sample_ties_of_the_first_rows(ops, vocab, kind):  # noqa: F811
    """A border among the first rows, which share a score: by top-k and top-p in a list, by top-p alone."""
    rng = rng_for("first ties", vocab, kind)
    z = -9 + rng.rand(vocab)
    z[rng.permutation(np.arange(200, vocab))[:280]] = 1.5 + rng.rand(280)
    z[:100] = 1.0
    scores = cuda(z[None].astype(np.float32), TYPES[kind])
    z = f64(scores)[0]
    w = np.exp(z - z.max())
    high, tie = w[z > 1].sum(), w[0]
    ties = np.repeat([1, 2, 7, 33, 64, 99], 4)              # how many of the equal ones remain
    n = len(ties)
    u = np.tile([0.0, 0.1, 0.6, 1 - 2.0 ** -24], n // 4).astype(np.float32)
    scores = scores.expand(n, vocab)
    sample_check(ops, scores, u, top_k=(280 + ties).astype(np.int32))
    listed = np.full(n, 380, np.int32)
    sample_check(ops, scores, u, top_k=listed, top_p=((high + (ties - 0.5) * tie) / (high + 100 * tie)).astype(np.float32))
    sample_check(ops, scores, u, top_p=((high + (ties - 0.5) * tie) / w.sum()).astype(np.float32))


@pytest.mark.parametrize("vocab", [20, 5000, 131072])
def test_sample_logp_of_unlikely_rows(ops, vocab):  # noqa: F811
    """The log-probability of a row far below the best is rounded to float32 and not to the steps of the sums."""
    n = 30
    z = np.full((n, vocab), -100.0)
    z[:, 0] = -0.9 * (np.arange(n) + 1) + 1 / 3             # down to 2^-38.5 of the best
    z[:, 7] = 0.0
    z[:, 11] = -0.5
    for kw in ({}, {"top_k": 3}, {"temperature": 0.97, "top_p": 1.0, "min_p": 0.0}):
        got = sample_check(ops, cuda(z.astype(np.float32)), np.zeros(n, np.float32), **kw)
        assert (got == 0).all()


# ---------------------------------------------------------------- lookups in a store
@pytest.mark.parametrize("storage", ["f32", "bf16"])
@pytest.mark.parametrize("end", ["close", "grow"])
def test_store_waits_for_lookups(ops, storage, end):  # noqa: F811
    """A store that gives its rows' memory back, because it is closed or its rows move, first waits for the lookups that read it,
    on whatever streams they are."""
    from vectordb_amd import _native
    x = rng_for("store", storage).randn(3000, 64).astype(np.float32)
    kept = cuda(x) if storage == "f32" else cuda(x).bfloat16().float()
    a = torch.randn(4096, 4096, device="cuda")
    rows = torch.arange(3000, device="cuda").repeat(20)
    streams = [torch.cuda.Stream(), torch.cuda.Stream(), torch.cuda.Stream()]
    for s in streams:                                      # libraries and streams made ready beforehand
        with torch.cuda.stream(s):
            a @ a
    store = _native.RowStore(64, storage=storage)
    store.append(x)
    torch.cuda.synchronize()
    got = []
    for s in streams:
        with torch.cuda.stream(s):
            b = a
            for _ in range(40):                            # some milliseconds of work before the lookup
                b = b @ a
            got.append(ops.lookup(store, rows, scale=0.5))
    if end == "close":
        store.close()
    else:
        store.append(np.zeros((200_000, 64), np.float32))
    done = [s.query() for s in streams]
    torch.cuda.synchronize()
    assert all(done)
    for g in got:
        assert torch.equal(g, 0.5 * kept[rows])
    store.close()


# ---------------------------------------------------------------- gradient of a lookup: tables as large as are allowed
def test_lookup_grad_largest_tables(ops):  # noqa: F811
    """More table rows to zero than a launch holds threads for, with no positions and with more than a quarter as many."""
    n_rows = 2 ** 30 - 1
    out = torch.full((n_rows, 1), 7.0, device="cuda", dtype=torch.bfloat16)
    none = torch.zeros(0, device="cuda", dtype=torch.int64)
    ops.lookup_grad(torch.zeros(0, 1, device="cuda", dtype=torch.bfloat16), none, n_rows, out=out)
    assert int((out != 0).sum()) == 0
    n = 2 ** 28 + 7
    out.fill_(7.0)
    rows = torch.arange(n, device="cuda") * 3 + 5            # every third row once, from the sixth on
    ops.lookup_grad(torch.ones(1, 1, device="cuda", dtype=torch.bfloat16).expand(n, 1), rows, n_rows, scale=3.0, out=out)
    named = torch.zeros(n_rows, device="cuda", dtype=torch.bool)
    named[rows] = True
    assert int((out[:, 0] != 3.0 * named).sum()) == 0


# ---------------------------------------------------------------- sampling: long rows that neither a list nor one bin settles
@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_sample_rows_without_outliers(ops, kind):  # noqa: F811
    """131072 scores of standard deviation 1: borders in the bulk, where a bin or a list is too small for those at the border."""
    rng = rng_for("bulk", kind)
    z = cuda(rng.randn(3, 131_072).astype(np.float32), TYPES[kind])
    u = np.array([0.02, 0.5, 0.97], np.float32)
    for kw in ({"temperature": 2.0, "top_p": 0.5}, {"temperature": 2.0, "top_p": 0.9}, {"temperature": 3.0, "min_p": 0.02}, {"min_p": 0.1}, {"top_k": 5000},
               {"top_k": 1025, "top_p": 0.5}, {"top_p": 0.3, "min_p": 0.05}):
        sample_check(ops, z, u, **kw)


# ---------------------------------------------------------------- distillation from a search
@pytest.mark.parametrize("n_rows", [7, 2000])
def test_distill_from_a_search(ops, n_rows):  # noqa: F811
    """The lists of a search as a teacher: distances, negated, with slots that a small store cannot fill."""
    from vectordb_amd import _native
    rng = rng_for("search", n_rows)
    x, q, k = rng.randn(n_rows, 48).astype(np.float32), rng.randn(9, 48).astype(np.float32), 10
    store = _native.RowStore(48)
    store.append(x)
    queries = cuda(q)
    dist, rows = torch.empty(9, k, device="cuda"), torch.empty(9, k, dtype=torch.int64, device="cuda")
    store.search_device(queries.data_ptr(), 9, k, _native.METRIC_CODES["euclidean"], dist.data_ptr(), rows.data_ptr(),
                        stream=torch.cuda.current_stream().cuda_stream)
    scores = torch.randn(9, n_rows, device="cuda")
    loss, stats = ops.distill(scores, -dist, rows)
    grad = ops.distill_grad(scores, -dist, rows, stats, torch.ones(9, device="cuda"))
    assert bool((rows < 0).any()) == (n_rows < k)
    for i in range(9):
        r = R.distill_row(f64(scores[i]), f64(-dist[i]), rows[i].cpu().numpy(), 1.0)
        # sums of 2000 / 256 terms a thread and of ten slots, exponents up to 10: 200 roundings cover them
        assert abs(float(loss[i]) - r["loss"]) <= 200 * U * max(1.0, abs(r["loss"]))
        assert (np.abs(f64(grad[i]) - r["grad"]) <= 200 * U * (r["q"] + r["target"])).all()
    store.close()
