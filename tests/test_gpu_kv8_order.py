"""Order between threads, products and kernels of the 8-bit cache and the
logit scores: calls whose warps, tiles or clusters finish apart give the same
bits every time, and the right ones."""
import numpy as np
import pytest

import hotseat_b200 as hs
from test_gpu_kv8 import check_rows, filled, i32, rows_of

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("nh, nkv, hd, n", [(14, 2, 64, 2048), (7, 1, 64, 1300), (5, 1, 128, 1100), (12, 2, 128, 20000)])
def test_single_rows_whose_shares_leave_lanes_idle(dtype, nh, nkv, hd, n):
    """A cluster's share of the outputs is no multiple of a warp: 7 columns of 64 in 8 shares are 14 pieces each."""
    rng = np.random.default_rng(n)
    kvs, refs = filled(rng, [n, n - 500], nkv, hd, 1, 0)
    s = hs.Kv8Set(kvs, n_heads=nh)
    q, qf = rows_of(rng, 2, nh, hd, dtype)
    pos, first = i32([n - 1, n - 501]), None
    for _ in range(40):
        out = torch.full_like(q, 9.0)
        s.attend(0, q, out, pos)
        first = out if first is None else first
        assert torch.equal(out, first)
    check_rows(first.float().cpu().numpy(), qf, refs, [(0, n - 1), (1, n - 501)], hd ** -0.5, dtype)


@pytest.mark.parametrize("rows, vocab, top", [(1, 151936, 5), (3, 40000, 20), (40, 20000, 3), (80, 9000, 64)])
def test_logit_scores_of_a_cluster_repeat(rows, vocab, top):
    g = torch.Generator(device="cuda").manual_seed(rows)
    x = torch.randn(rows, vocab, generator=g, device="cuda") * 3
    ids = torch.randint(0, vocab, (rows,), generator=g, device="cuda", dtype=torch.int32)
    first = None
    for _ in range(40):
        o = dict(logp=torch.empty(rows, device="cuda"), entropy=torch.empty(rows, device="cuda"),
                 rank=torch.empty(rows, dtype=torch.int32, device="cuda"),
                 top_ids=torch.empty(rows, top, dtype=torch.int32, device="cuda"),
                 top_logp=torch.empty(rows, top, device="cuda"))
        hs.logprobs(x, ids, **o)
        first = first or o
        assert all(torch.equal(o[k], first[k]) for k in o)
    want = torch.log_softmax(x.double(), -1).gather(1, ids.long()[:, None])[:, 0]
    assert float((first["logp"] - want).abs().max()) <= 64 * 2.0 ** -24 * float(want.abs().max())
    assert torch.equal(first["top_ids"].long(), torch.sort(x, dim=-1, descending=True, stable=True).indices[:, :top])


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("nh, nkv, hd, block", [(14, 2, 64, 16), (12, 2, 128, 1)])
def test_chunks_repeat_over_many_tiles(dtype, nh, nkv, hd, block):
    """Prompts, one row tile alone and rows that a cluster shares: each tile's scores take the place of the weights
    that the product before them read."""
    rng = np.random.default_rng(hd)
    lens, rows = [1500, 2000, 700, 5000], [300, 40, 700, 9]
    kvs, refs = filled(rng, lens, nkv, hd, block, 0)
    s = hs.Kv8Set(kvs, n_heads=nh)
    start = np.concatenate([[0], np.cumsum(rows)])
    q, qf = rows_of(rng, sum(rows), nh, hd, dtype)
    pos, start_d, first = i32([n - m for n, m in zip(lens, rows)]), i32(start), None
    for _ in range(20):
        out = torch.full_like(q, 9.0)
        s.attend(0, q, out, pos, start_d)
        first = out if first is None else first
        assert torch.equal(out, first)
    s.check()
    places = [(i, n - m + j) for i, (n, m) in enumerate(zip(lens, rows)) for j in range(m)]
    pick = [0, 299, 300, 339, 340, 700, 1039, 1040, 1048]
    check_rows(first.float().cpu().numpy()[pick], qf[pick], refs, [places[i] for i in pick], hd ** -0.5, dtype)


@pytest.mark.parametrize("block, layout, hd", [(1, 0, 64), (16, 0, 64), (16, 1, 128), (64, 1, 64), (128, 0, 128)])
def test_a_pre_copy_beside_appends_misses_nothing(block, layout, hd):
    """Armed, harvested and copied while appends run on another stream: once these are done, one more harvest makes
    the copy equal. Half steps keep a row's lanes apart."""
    rng = np.random.default_rng(block)
    spec = hs.KvSpec(1, 2, hd, 1024, layout)
    src, dst = hs.Kv.alloc8(spec, block=block, page_size=256), hs.Kv.alloc8(spec, block=block, page_size=256)
    s, side = hs.Kv8Set([src]), torch.cuda.Stream()
    x = rng.integers(-126, 126, (1024, 2, hd)) + np.where(rng.random((1024, 2, hd)) < 0.1, 0.5, 0.0)
    x[..., 0] = 127.0
    x = x * 2.0 ** rng.integers(0, 3, (1024, 1, 1))
    k = torch.from_numpy(x.astype(np.float32)).cuda()
    starts, sizes = [], []
    p = 0
    while p < 1024:
        m = min(int(rng.integers(1, 9)), 1024 - p)
        starts.append(i32([p]))
        sizes.append((p, m, i32([0, m])))
        p += m
    torch.cuda.synchronize()
    at = 0

    def some(n):
        nonlocal at
        for pos, (p, m, row) in zip(starts[at:at + n], sizes[at:at + n]):
            s.append(0, k[p:p + m], k[p:p + m], pos, row, stream=side.cuda_stream)
        at += n

    whole = [(0, src.bytes)]
    some(20)
    src.arm()
    src.copy_runs_to(dst, whole)
    while at < len(starts):
        some(12)
        words = src.harvest()
        src.copy_runs_to(dst, hs.runs_to_byte_runs(words, src.n_pages, src.page_size, whole))
    side.synchronize()
    src.copy_runs_to(dst, hs.runs_to_byte_runs(src.harvest(), src.n_pages, src.page_size, whole))
    assert np.array_equal(src.read(0, src.bytes), dst.read(0, dst.bytes))
    src.disarm()
    s.check()
