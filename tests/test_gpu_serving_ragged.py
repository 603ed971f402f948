"""Batches whose bounds lie far above most of their sequences: a few prompts among many entries."""
import numpy as np
import pytest

from conftest import bf16_bits, bf16_vals
from serving_kit import Cache, Device, attention64, attention_bounds

pytestmark = pytest.mark.gpu

BAD_BATCH = 5


@pytest.mark.parametrize("grouped", [False, True])
def test_wide_bounds_over_many_entries(tiny_model, grouped):
    """512 entries, a million tokens and 128 rows as the bounds of one: what the bounds multiply to says nothing about the work, which is two
    prompts of 128 rows and a few single rows among entries of -1."""
    from q3asr import AttentionBatch
    heads, dim, pg, width, n = 8, 64, 256, 4096, 512
    with Device() as dev:
        c = Cache(dev, tiny_model[0], seqs=n, width=width, pages=16, heads=heads, dim=dim, pg=pg, seed=4)
        rng = np.random.default_rng(4)
        real = {3: (128, 128), 100: (300, 1), 101: (517, 128), 400: (1, 1), 511: (256, 2)}      # entry: tokens, rows
        seqs, rows = [-1] * n, [0] * n
        for s, (e, (_, r)) in enumerate(real.items()):
            seqs[e], rows[e] = 7 * s + 2, r
        c.reserve([seqs[e] for e in real], [t for t, _ in real.values()])
        cu = np.concatenate([[0], np.cumsum(rows)]).tolist()
        kw = dict(seqs=c.ints(seqs), cu_rows=c.ints(cu), n=n, rows=cu[-1], max_rows=128, max_len=width * pg)
        if grouped:
            kw.update(cu_groups=c.ints(range(0, n + 1, 4)), shared=c.ints([0] * (n // 4)), n_groups=n // 4, max_group_rows=129, max_shared=width * pg,
                      max_own=width * pg)
        q = bf16_bits(rng.standard_normal((cu[-1], heads * dim)))
        b = AttentionBatch(**kw)
        at, nb = dev.put(q), c.c.attention_workspace_bytes(b, heads)
        o, e = dev.raw(q.nbytes), dev.raw(4 * cu[-1] * heads)
        c.c.attention(0, at, o, b, heads, lse=e, workspace=(dev.raw(nb), nb))
        got = bf16_vals(dev.get(o, q.shape, np.uint16)).astype(np.float64).reshape(-1, heads, dim)
        for i in real:
            k, v = c.book.keys(0, seqs[i])
            x = bf16_vals(q[cu[i]:cu[i + 1]]).astype(np.float64).reshape(-1, heads, dim)
            want, _, size, slack = attention64(x, k, v, c.book.lens[seqs[i]], rows[i], heads, dim ** -0.5)
            assert (np.abs(got[cu[i]:cu[i + 1]] - want) <= attention_bounds(want, size, slack, c.book.lens[seqs[i]])).all(), i


@pytest.mark.parametrize("over", ["cu_rows", "cu_groups"])
@pytest.mark.parametrize("n", [100, 1500])
def test_lists_that_go_down_are_reported_and_write_nothing(tiny_model, over, n):
    """cu_rows that names the same rows for every second entry, cu_groups that names the same entries for every second group."""
    from q3asr import AttentionBatch
    heads, dim, pg = 2, 64, 16
    with Device() as dev:
        c = Cache(dev, tiny_model[0], seqs=n, width=66, pages=2 * n, heads=heads, dim=dim, pg=pg, seed=4)
        c.reserve(list(range(n)), [20] * n)
        lists = dict(cu_rows=list(range(0, 8 * n + 1, 8)), cu_groups=list(range(0, n + 1, 2)))
        top = lists[over][-1]
        lists[over] = [(0, top)[i % 2] for i in range(len(lists[over]))]
        b = AttentionBatch(seqs=c.ints(range(n)), n=n, rows=8 * n, max_rows=8 * n, max_len=1056, shared=c.ints([16] * (n // 2)), n_groups=n // 2,
                           max_group_rows=8 * n, max_shared=16, max_own=1056, **{k: c.ints(v) for k, v in lists.items()})
        q = dev.put(bf16_bits(np.ones((8 * n, heads * dim))))
        o, nb, st = dev.put(np.full((8 * n, heads * dim), 7, np.uint16)), c.c.attention_workspace_bytes(b, heads), dev.stream()
        c.c.attention(0, q, o, b, heads, workspace=(dev.raw(nb), nb), stream=st)
        assert c.c.status(stream=st)[0] == BAD_BATCH
        assert (dev.get(o, (8 * n, heads * dim), np.uint16) == 7).all()


def test_runs_past_32_bits(tiny_model):
    """Entries times layers times KV heads past 2^32: the copies' grid is counted in 64 bits.  No page is shared and none lies behind a gap, so
    nothing is copied and the pools are never touched."""
    from q3asr import PagedKVCache
    n = 1024
    with Device() as dev:
        pool = dev.raw(16)
        at = {"table": dev.raw(4 * n * 2), "lens": dev.raw(4 * n), "refs": dev.raw(4 * n), "status": dev.raw(16)}
        c = PagedKVCache(tiny_model[0], k=pool, v=pool, layers=4096, pages=n, kv_heads=4096, head_dim=64, page_tokens=16, max_seqs=n, max_seq_pages=2, **at)
        nb = c.workspace_bytes()
        c.set_workspace(dev.raw(nb), nb)
        c.reset()
        c.reserve(dev.put(np.arange(n, dtype=np.int32)), dev.put(np.full(n, 3, np.int32)), n)
        c.compact()
        assert c.status()[:3] == (0, 0, 0)
        assert np.array_equal(dev.get(at["table"], (n, 2), np.int32), np.stack([np.arange(n), np.full(n, -1)], 1))
        assert (dev.get(at["lens"], n, np.int32) == 3).all() and (dev.get(at["refs"], n, np.int32) == 1).all()
