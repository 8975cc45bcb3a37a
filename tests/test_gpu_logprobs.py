"""Scores of logit rows against 64 bits. Bounds: a log probability is
x - m - ln l with m exact, l a sum of exponentials each off by a few u
relatively (u = 2^-24; the argument of an exponential up to A = max - x
rounds by A u, so a term e^-A by A u e^-A, at most u), and its log; so
8 u + 2 u (|x - m| + ln l). Entropy adds the mean of (x - m), as large as the
spread of what has weight: 16 u (1 + entropy + ln vocab)."""
import numpy as np
import pytest

import hotseat_b200 as hs

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
U = 2.0 ** -24


def run(x, ids, top):
    rows = x.shape[0]
    o = dict(logp=torch.empty(rows, device="cuda"), entropy=torch.empty(rows, device="cuda"),
             rank=torch.empty(rows, dtype=torch.int32, device="cuda"),
             top_ids=torch.full((rows, top), -7, dtype=torch.int32, device="cuda"),
             top_logp=torch.empty(rows, top, device="cuda"))
    hs.logprobs(x, ids, **o)
    return {k: v.cpu().numpy() for k, v in o.items()}


def order(row):
    """Token ids, first to last: value descending (NaN first, -0 as 0), id ascending."""
    key = np.where(np.isnan(row), np.inf, row + 0.0)
    return np.lexsort((np.arange(row.size), -key, ~np.isnan(row)))


def check(x, ids, top):
    got = run(x, ids, top)
    v = x.float().cpu().numpy().astype(np.float64)
    ids = ids.cpu().numpy()
    for r in range(v.shape[0]):
        row = v[r]
        by = order(row)
        assert got["top_ids"][r].tolist() == by[:top].tolist()
        t = int(ids[r])
        if 0 <= t < row.size:
            assert got["rank"][r] == int(np.nonzero(by == t)[0][0])
        else:
            assert got["rank"][r] == -1 and np.isnan(got["logp"][r])
        with np.errstate(all="ignore"):
            m = row.max()
            if not np.isfinite(m):
                assert np.isnan(got["entropy"][r]) and np.isnan(got["top_logp"][r]).all() and np.isnan(got["logp"][r])
                continue
            e = np.exp(row - m)
            lz = np.log(e.sum())
            lp = row - m - lz
            p = e / e.sum()
            ent = -np.sum(np.where(p > 0, p * np.where(p > 0, lp, 0), 0))
        def near(a, i):
            if np.isneginf(lp[i]):
                return np.isneginf(a)
            return abs(a - lp[i]) <= 8 * U + 2 * U * (abs(row[i] - m) + lz) + U * abs(lp[i])
        if 0 <= t < row.size:
            assert near(got["logp"][r], t), (got["logp"][r], lp[t])
        for j in range(top):
            assert near(got["top_logp"][r][j], by[j])
        assert abs(got["entropy"][r] - ent) <= 16 * U * (1 + ent + np.log(row.size)), (got["entropy"][r], ent)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows, vocab, top", [(1, 1, 1), (3, 2, 2), (2, 33, 33), (5, 1000, 20), (2, 4097, 64),
                                              (3, 20011, 5), (4, 151936, 20), (1, 151936, 64), (2, 500000, 7)])
def test_rows_of_every_length(dtype, rows, vocab, top):
    g = torch.Generator(device="cuda").manual_seed(rows + vocab)
    x = (torch.randn(rows, vocab, generator=g, device="cuda") * 4).to(DT[dtype])
    ids = torch.randint(0, vocab, (rows,), generator=g, device="cuda", dtype=torch.int32)
    check(x, ids, top)


@pytest.mark.parametrize("top", [0, 1, 17, 64])
def test_ties_go_to_the_lowest_id(top):
    rng = np.random.default_rng(top)
    x = torch.from_numpy(rng.integers(-2, 3, size=(6, 9001)).astype(np.float32)).cuda()
    x[0] = 1.0
    x[1, ::2] = -0.0
    x[1, 1::2] = 0.0
    x[2] = torch.arange(9001, device="cuda")
    x[3] = -torch.arange(9001, device="cuda").float()
    ids = torch.tensor([9000, 4, 0, 9000, 17, 8999], dtype=torch.int32, device="cuda")
    check(x, ids, top)


def test_masked_rows():
    inf, nan = float("inf"), float("nan")
    x = torch.randn(9, 3001, device="cuda", generator=torch.Generator(device="cuda").manual_seed(1))
    x[0, 100:] = -inf                      # most of the row cannot come
    x[1, :] = -inf
    x[1, 1234] = 2.0                       # one token left: certain
    x[2, :] = -inf                         # none left
    x[3, 7] = inf
    x[4, 9] = nan
    x[4, 3] = nan
    x[5, :] = torch.finfo(torch.float32).min
    x[5, 50] = 0.0
    x[6, :] = torch.finfo(torch.float32).min
    x[7, ::3] = -inf
    x[8, :] = nan
    ids = torch.tensor([5, 1234, 0, 7, 3, 50, 2, 0, 2999], dtype=torch.int32, device="cuda")
    check(x, ids, 20)
    ids = torch.tensor([2000, 0, 3000, 0, 0, 3, 3000, 3000, 0], dtype=torch.int32, device="cuda")
    check(x, ids, 1)


def test_ids_outside_the_vocabulary():
    x = torch.randn(3, 77, device="cuda")
    check(x, torch.tensor([77, -1, 3], dtype=torch.int32, device="cuda"), 4)


def test_outputs_that_are_not_wanted_and_strided_rows():
    g = torch.Generator(device="cuda").manual_seed(4)
    wide = torch.randn(5, 1003, generator=g, device="cuda")
    for x in (wide[:, 1:1000], wide[::2, 3:900], wide[:, :999]):
        ids = torch.arange(x.shape[0], dtype=torch.int32, device="cuda")
        check(x, ids, 9)
    for dt in (torch.float16, torch.bfloat16):
        check(wide.to(dt)[:, 1:1000], torch.arange(5, dtype=torch.int32, device="cuda"), 9)
    full = run(wide, torch.zeros(5, dtype=torch.int32, device="cuda"), 6)
    ent, ids6 = torch.empty(5, device="cuda"), torch.empty(5, 6, dtype=torch.int32, device="cuda")
    hs.logprobs(wide, entropy=ent)
    hs.logprobs(wide, top_ids=ids6)
    assert np.array_equal(ent.cpu().numpy(), full["entropy"]) and np.array_equal(ids6.cpu().numpy(), full["top_ids"])
    rank = torch.empty(5, dtype=torch.int32, device="cuda")
    hs.logprobs(wide, torch.zeros(5, dtype=torch.int32, device="cuda"), rank=rank)
    assert np.array_equal(rank.cpu().numpy(), full["rank"])
    hs.logprobs(wide[:0])


def test_a_rows_bits_do_not_depend_on_the_batch_or_the_call():
    x = torch.randn(300, 30011, device="cuda", generator=torch.Generator(device="cuda").manual_seed(9)) * 3
    ids = torch.arange(300, dtype=torch.int32, device="cuda") * 100
    a = run(x, ids, 8)
    for r in (0, 17, 299):
        b = run(x[r:r + 1], ids[r:r + 1], 8)
        assert all(np.array_equal(a[k][r:r + 1], b[k]) for k in a)
    out = torch.empty(300, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    hs.logprobs(x, ids, logp=out, stream=side.cuda_stream)
    side.synchronize()
    assert np.array_equal(out.cpu().numpy(), a["logp"])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        hs.logprobs(x, ids, logp=out, stream=side.cuda_stream)
    out.zero_()
    graph.replay()
    torch.cuda.synchronize()
    assert np.array_equal(out.cpu().numpy(), a["logp"])


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("vocab, top", [(9001, 64), (70003, 5), (200011, 20)])
def test_many_rows_have_the_bits_of_few(dtype, vocab, top):
    """Up to 600 rows at once against the same rows in calls of 12: plain ones, logits in order either way, ties, masked
    rows with and without enough tokens left, NaN."""
    inf, nan = float("inf"), float("nan")
    g = torch.Generator(device="cuda").manual_seed(vocab)
    some = torch.randn(12, vocab, generator=g, device="cuda") * 3
    some[1] = torch.arange(vocab, device="cuda") / vocab * 8
    some[2] = -some[1]
    some[3] = torch.randint(-2, 3, (vocab,), generator=g, device="cuda").float()
    some[4, :-3] = -inf
    some[5] = -inf
    some[6, 100:-100] = -inf
    some[7, -1] = nan
    some[8, ::2] = nan
    some[9, vocab // 2] = inf
    some[10, vocab // 2:] += 20.0
    some = some.to(DT[dtype])
    ids = torch.tensor([0, 5, vocab - 1, 77, vocab - 2, 3, 50, 9, 11, 4, vocab - 1, -1], dtype=torch.int32, device="cuda")
    check(some, ids, top)
    few = run(some, ids, top)
    for times in (50, 26, 13):
        many = run(some.repeat(times, 1), ids.repeat(times), top)
        for k in few:
            want = np.tile(few[k], (times,) + (1,) * (few[k].ndim - 1))
            assert np.array_equal(many[k], want, equal_nan=want.dtype == np.float32), (k, times)


@pytest.mark.parametrize("dtype", ["f32", "f16"])
def test_many_rows_off_their_alignment(dtype):
    """Rows that begin one element past an aligned place, in one call of 600 and in small ones."""
    g = torch.Generator(device="cuda").manual_seed(5)
    x = (torch.randn(600, 9003, generator=g, device="cuda") * 4).to(DT[dtype])[:, 1:]
    ids = torch.randint(0, 9002, (600,), generator=g, device="cuda", dtype=torch.int32)
    many = run(x, ids, 33)
    check(x[590:], ids[590:], 33)
    for at in (0, 299, 590):
        few = run(x[at:at + 10], ids[at:at + 10], 33)
        assert all(np.array_equal(many[k][at:at + 10], few[k]) for k in few)


def test_scores_of_a_forward(tiny_gguf):
    m = hs.Model.load(tiny_gguf, max_ctx=16)
    s, kv = m.scratch(), m.kv()
    m.forward(kv, 5, 0, s)
    got, row = s.logprobs(17, top=5), s.logits().astype(np.float64)
    lz = np.log(np.exp(row - row.max()).sum()) + row.max()
    assert abs(got["logp"] + s.nll(17)) <= 1e-5 and abs(got["logp"] - (row[17] - lz)) <= 1e-5
    assert got["top_ids"].tolist() == order(row)[:5].tolist()
    assert int(got["rank"]) == int(np.nonzero(order(row) == 17)[0][0])
    with pytest.raises(hs.HotseatError):
        s.logprobs(m.cfg.vocab)
    t = hs.Model.load(tiny_gguf, max_ctx=16, numeric=hs.NUMERIC_TC)
    b, kvs = hs.Batch(t, 3), [t.kv() for _ in range(3)]
    b.forward(kvs, [5, 6, 7], [0, 0, 0])
    o, nll = b.logprobs([1, 2, 3], top=4), b.nll([1, 2, 3])
    assert np.all(np.abs(o["logp"] + nll) <= 1e-5)
    for i in range(3):
        assert o["top_ids"][i].tolist() == order(b.logits(i).astype(np.float64))[:4].tolist()
    o = b.logprobs([4, 5])
    assert o["top_ids"].shape == (2, 0) and np.all(np.abs(o["logp"] + b.nll([4, 5])) <= 1e-5)
    with pytest.raises(hs.HotseatError):
        b.logprobs([m.cfg.vocab])
