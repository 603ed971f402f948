"""Attention over the paged cache against 64-bit arithmetic, and a decode step of several hypotheses from all serving operators."""
import numpy as np
import pytest

from conftest import bf16_bits, bf16_vals
from q3asr.lib import Q3Error
from serving_kit import F32_HALF_STEP, Cache, Device, attention64, attention_bounds

pytestmark = pytest.mark.gpu


class Step:
    """A cache with groups of sequences that share prefixes, and one step's rows."""

    def __init__(self, dev, model, groups, heads, kv, dim, pg, seed, poison=True, layers=2, layer=1, spread=1.0, spare=0):
        """groups: [(shared tokens, [(own tokens, rows), ...]), ...]; own tokens include the rows."""
        self.rng = rng = np.random.default_rng(seed)
        self.dev, self.heads, self.kv, self.dim, self.layer = dev, heads, kv, dim, layer
        members = [m for _, ms in groups for m in ms]
        n = len(members)
        lens = [s + own for s, ms in groups for own, _ in ms]
        width = max(1, -(-max(max(lens), 1040) // pg)) + 1
        pages = sum(-(-x // pg) + 1 for x in lens) + sum(s // pg + 2 for s, _ in groups) + 3
        self.c = c = Cache(dev, model, seqs=n + len(groups) + spare, width=width, pages=pages, layers=layers, heads=kv, dim=dim, pg=pg, seed=seed, poison=poison)
        # every group grows from a base sequence, pages scattered over the pool by a few that come and go
        first = 0
        self.shared, self.seqs, self.cu_groups = [], [], [0]
        for g, (s, ms) in enumerate(groups):
            base, own = n + g, list(range(first, first + len(ms)))
            c.book.reserve([base], [s])
            self._fill(base, 0, s)
            c.book.fork(own, [base] * len(ms))
            c.book.fork([base], [-1])
            c.book.reserve(own, [o for o, _ in ms])
            for q, (o, _) in zip(own, ms):
                self._fill(q, s, s + o)
            first += len(ms)
            self.seqs += own
            self.shared.append(s)
            self.cu_groups.append(first)
        c.put()
        dev.put(c.book.k, c.at["k"])
        dev.put(c.book.v, c.at["v"])
        self.rows = [r for _, ms in groups for _, r in ms]
        self.cu = np.concatenate([[0], np.cumsum(self.rows)]).tolist()
        self.lens = lens
        self.q = bf16_bits(rng.standard_normal((self.cu[-1], heads * dim)) * spread)

    def _fill(self, s, a, b):
        book = self.c.book
        for pos in range(a, b):
            p = book.tables[s][pos // book.pg]
            for pool in (book.k, book.v):
                pool[:, p, :, pos % book.pg] = bf16_bits(self.rng.standard_normal((pool.shape[0], pool.shape[2], pool.shape[4])))

    def batch(self, grouped=True, **over):
        from q3asr import AttentionBatch
        pg = self.c.book.pg
        kw = dict(seqs=self.c.ints(self.seqs), cu_rows=self.c.ints(self.cu), n=len(self.seqs), rows=self.cu[-1], max_rows=max(1, max(self.rows)),
                  max_len=max(self.lens))
        if grouped:
            cg = self.cu_groups
            kw.update(cu_groups=self.c.ints(cg), shared=self.c.ints(self.shared), n_groups=len(self.shared),
                      max_group_rows=max(self.cu[b] - self.cu[a] for a, b in zip(cg, cg[1:])), max_shared=max(self.shared),
                      max_own=max(n - s // pg * pg for s, a, b in zip(self.shared, cg, cg[1:]) for n in self.lens[a:b]))
        kw.update(over)
        return AttentionBatch(**kw)

    def run(self, batch, stream=None, pad=0, lse=True, scale=None, extra_rows=0):
        d, rows, width = self.dev, self.cu[-1], self.heads * self.dim
        ld = width + pad
        q = np.full((rows, ld), 0x7FC1, np.uint16)
        q[:, :width] = self.q
        o = d.put(np.full((rows + extra_rows, ld), 7, np.uint16))
        e = d.put(np.full((rows + extra_rows, self.heads), 7, np.float32))
        n = self.c.c.attention_workspace_bytes(batch, self.heads)
        self.c.c.attention(self.layer, d.put(q), o, batch, self.heads, scale=scale, q_ld=ld, o_ld=ld, lse=e if lse else None,
                           workspace=(d.put(np.full(max(n, 16), 0xFF, np.uint8)), n), stream=stream)
        if stream:
            d.wait(stream)
        out = d.get(o, (rows + extra_rows, ld), np.uint16)
        assert (out[:, width:] == 7).all() and (out[rows:] == 7).all()
        return out[:rows, :width], d.get(e, (rows + extra_rows, self.heads), np.float32)[:rows]

    def check(self, out, lse, scale=None):
        scale = self.dim ** -0.5 if scale is None else scale
        for i, s in enumerate(self.seqs):
            a, b = self.cu[i], self.cu[i + 1]
            k, v = self.c.book.keys(self.layer, s)
            q = bf16_vals(self.q[a:b]).astype(np.float64).reshape(b - a, self.heads, self.dim)
            want, want_lse, size, slack = attention64(q, k, v, self.lens[i], b - a, self.heads, scale)
            got = bf16_vals(out[a:b]).astype(np.float64).reshape(want.shape)
            assert np.isfinite(got).all(), (i, s)
            tol = attention_bounds(want, size, slack, self.lens[i])
            assert (np.abs(got - want) <= tol).all(), (i, s, (np.abs(got - want) / tol).max())
            seen = np.isfinite(want_lse)
            assert (lse[a:b][~seen] == -np.inf).all()
            bound = slack + (self.lens[i] + 64) * 2 * F32_HALF_STEP + 4 * F32_HALF_STEP * np.abs(np.where(seen, want_lse, 0))
            assert (np.abs(np.where(seen, lse[a:b] - np.where(seen, want_lse, 0), 0)) <= bound).all(), (i, s)


GROUPS = [
    [(0, [(1, 1)])],                                                             # one key
    [(5, [(1, 1), (1, 1)]), (16, [(1, 1)]), (0, [(17, 1)])],                     # shared less than a page, exactly one, nothing
    [(405, [(1, 1), (40, 1), (448, 1), (16, 1), (3, 1)])],
    [(33, [(70, 1)] * 3), (128, [(1, 1), (2, 1)]), (700, [(9, 1)] * 9), (64, [(600, 1)])],
    [(1600, [(5, 1)] * 4), (513, [(600, 1), (1, 1)])],                            # several chunks of either kind
    [(48, [(20, 20), (3, 1), (7, 7), (1, 1)]), (0, [(9, 9)]), (200, [(130, 64), (64, 2)])],   # several rows per sequence
    [(30, [(4, 0), (5, 1)]), (50, [(2, 2), (3, 0)])],                             # sequences without a row
]


@pytest.mark.parametrize("heads,kv,dim,pg", [(4, 2, 128, 16), (3, 3, 64, 32), (8, 1, 128, 64), (14, 2, 64, 16), (40, 2, 128, 16)])
@pytest.mark.parametrize("g", range(len(GROUPS)))
def test_attention_matches_fp64(tiny_model, g, heads, kv, dim, pg):
    with Device() as dev:
        s = Step(dev, tiny_model[0], GROUPS[g], heads, kv, dim, pg, seed=g)
        s.check(*s.run(s.batch(), pad=8 * (g % 2), extra_rows=1))
        s.check(*s.run(s.batch(grouped=False)))
        # a bound above 1024 tokens takes small steps, too, through the plan and the parts
        s.check(*s.run(s.batch(max_len=max(1040, max(s.lens))), pad=8, extra_rows=2))
        s.check(*s.run(s.batch(grouped=False, max_len=max(1040, max(s.lens)))))
        if g in (2, 5):      # bounds above what the batch needs, another scale, sharp rows, no lse
            m = (s.c.width - 1) * s.c.book.pg
            s.check(*s.run(s.batch(max_len=m, max_shared=m, max_own=m, max_group_rows=s.cu[-1])))
            s.check(*s.run(s.batch(), scale=0.9), scale=0.9)
            out, _ = s.run(s.batch(), lse=False)
            assert np.array_equal(out, s.run(s.batch())[0])
        assert s.c.c.status()[:3] == (0, 0, 0)


def test_more_sequences_than_a_workgroup_plans(tiny_model):
    """Over 1024 groups and sequences: planned by a launch of its own."""
    with Device() as dev:
        s = Step(dev, tiny_model[0], [(20, [(3, 1), (5, 2)])] * 400, 4, 2, 64, 16, seed=6)
        s.check(*s.run(s.batch()))
        s.check(*s.run(s.batch(grouped=False, max_len=1040)))
        assert s.c.c.status()[:3] == (0, 0, 0)


def test_long_sequences(tiny_model):
    """Tens of thousands of keys for one row and for a group: many parts, page windows that are renewed on the way."""
    with Device() as dev:
        s = Step(dev, tiny_model[0], [(0, [(21007, 1)]), (9000, [(40, 3), (1200, 1)])], 2, 1, 128, 32, seed=8)
        s.check(*s.run(s.batch()))


def test_padded_batches(tiny_model):
    """Entries of -1, sequences without rows and rows behind the last sequence's: left alone, nothing is reported."""
    with Device() as dev:
        for over in ({}, dict(max_len=1040)):
            s = Step(dev, tiny_model[0], [(40, [(3, 1), (9, 2)]), (64, [(30, 1)])], 4, 2, 128, 16, seed=12, spare=2)
            n, rows = 7, s.cu[-1] + 3
            real = s.cu[-1]
            seqs, cu, groups, shared = s.seqs + [-1] * 4, s.cu + [real] * 4, s.cu_groups + [5, 7], s.shared + [48, 0]
            s.q = np.concatenate([s.q, s.q[:3]])
            s.cu[-1] = rows                       # buffers of the padded size
            b = s.batch(seqs=s.c.ints(seqs), cu_rows=s.c.ints(cu), cu_groups=s.c.ints(groups), shared=s.c.ints(shared), n=n, rows=rows, n_groups=4,
                        max_rows=2, max_group_rows=4, max_own=max(s.lens), **over)
            out, lse = s.run(b)
            assert s.c.c.status()[:3] == (0, 0, 0)
            assert (out[real:] == 7).all() and (lse[real:] == 7).all()
            s.cu[-1] = real
            s.check(out[:real], lse[:real])


def test_rows_without_keys_are_zero(tiny_model):
    """Empty sequences and rows before a sequence's first token: zeros and -inf, with and without groups."""
    with Device() as dev:
        s = Step(dev, tiny_model[0], [(0, [(0, 0), (0, 0)]), (20, [(2, 1)])], 4, 2, 128, 16, seed=2)
        # sequence 0: no token, one row; sequence 1: no token, two rows
        s.rows, s.cu = [1, 2, 1], [0, 1, 3, 4]
        s.q = bf16_bits(s.rng.standard_normal((4, 512)))
        for b in (s.batch(), s.batch(grouped=False), s.batch(max_len=1040), s.batch(grouped=False, max_len=1040)):
            out, lse = s.run(b)
            s.check(out, lse)
            assert (out[:3] == 0).all() and (lse[:3] == -np.inf).all()
    with Device() as dev:      # more rows than tokens: the first ones lie before the sequence
        s = Step(dev, tiny_model[0], [(0, [(1, 1), (3, 3)])], 4, 2, 128, 16, seed=3)
        s.rows, s.cu = [3, 5], [0, 3, 8]
        s.q = bf16_bits(s.rng.standard_normal((8, 512)))
        for b in (s.batch(), s.batch(grouped=False, max_len=1040)):
            out, lse = s.run(b)
            s.check(out, lse)
            assert (out[[0, 1, 3, 4]] == 0).all() and np.isfinite(lse[[2, 5, 6, 7]]).all()


def test_extreme_scores(tiny_model):
    """One key far above the others in the last and in the first place, equal scores everywhere, scores of thousands."""
    with Device() as dev:
        s = Step(dev, tiny_model[0], [(100, [(60, 2), (9, 1)])], 4, 2, 128, 16, seed=4, spread=30.0)
        for b in (s.batch(), s.batch(max_len=1040)):
            s.check(*s.run(b))
        s.q[:] = 0                       # a flat softmax
        for b in (s.batch(), s.batch(max_len=1040)):
            s.check(*s.run(b))


@pytest.mark.parametrize("dim,heads,kv", [(128, 4, 2), (64, 14, 2)])
@pytest.mark.parametrize("scale", [0.125, -0.5, 0.0])
def test_scores_that_rise_along_the_keys(tiny_model, dim, heads, kv, scale):
    """Running maxima that move at every key, by little and by much, or never after the first key; scales of either sign and zero.
    Few sequences that are long enough for more parts than lanes take at once, and several rows per sequence."""
    for seed, step in enumerate((0.3, 9.0)):
        with Device() as dev:
            s = Step(dev, tiny_model[0], [(2600, [(70, 1), (300, 3), (5, 1)])], heads, kv, dim, 16, seed=seed)
            book = s.c.book
            for i, q in enumerate(s.seqs):   # values along one dimension grow with the position, in their own pages and in shared ones
                for pos in range(s.lens[i]):
                    book.k[:, book.tables[q][pos // book.pg], :, pos % book.pg, 3] = bf16_bits(np.array([step * pos / 8]))[0]
            dev.put(book.k, s.c.at["k"])
            for sign in (1, -1):
                s.q.reshape(len(s.q), heads, dim)[:, :, 3] = bf16_bits(np.array([float(sign)]))[0]
                for grouped in (True, False):
                    s.check(*s.run(s.batch(grouped), scale=scale), scale=scale)


@pytest.mark.parametrize("dim,kv", [(128, 8), (64, 2)])
def test_long_cache_past_32_bit_offsets(tiny_model, dim, kv):
    """A pool whose last pages lie behind 2^31 values."""
    from q3asr import AttentionBatch, PagedKVCache
    heads, pg = 2 * kv, 256
    pages = (1 << 31) // (kv * pg * dim) + 40
    rng = np.random.default_rng(1)
    with Device() as dev:
        pool = pages * kv * pg * dim
        at = {n: dev.raw(2 * pool) for n in "kv"}
        n, width = 700, 3
        use = [pages - 1, 2, pages - 3]
        page = kv * pg * dim
        data = {}
        for name in "kv":
            for p in use:
                data[name, p] = bf16_bits(rng.standard_normal((kv, pg, dim)))
                dev.put(data[name, p], at[name] + 2 * p * page)
        at.update(table=dev.put(np.array([use], np.int32)), lens=dev.put(np.array([n], np.int32)), refs=dev.put(np.zeros(pages, np.int32)),
                  status=dev.put(np.zeros(4, np.int32)))
        c = PagedKVCache(tiny_model[0], layers=1, pages=pages, kv_heads=kv, head_dim=dim, page_tokens=pg, max_seqs=1, max_seq_pages=width, **at)
        q = bf16_bits(rng.standard_normal((1, heads * dim)))
        b = AttentionBatch(seqs=dev.put(np.zeros(1, np.int32)), cu_rows=dev.put(np.array([0, 1], np.int32)), n=1, rows=1, max_rows=1, max_len=n)
        o, e, ws = dev.raw(2 * heads * dim), dev.raw(4 * heads), c.attention_workspace_bytes(b, heads)
        c.attention(0, dev.put(q), o, b, heads, lse=e, workspace=(dev.raw(ws), ws))
        k, v = (np.concatenate([bf16_vals(data[x, p]) for p in use], 1)[:, :n].astype(np.float64) for x in "kv")
        want, want_lse, size, slack = attention64(bf16_vals(q).astype(np.float64).reshape(1, heads, dim), k, v, n, 1, heads, dim ** -0.5)
        got = bf16_vals(dev.get(o, (1, heads, dim), np.uint16)).astype(np.float64)
        assert (np.abs(got - want) <= attention_bounds(want, size, slack, n)).all()


def test_wrong_batches_are_reported(tiny_model):
    """What the device finds wrong is reported, stays inside the buffers and leaves the cache usable."""
    with Device() as dev:
        s = Step(dev, tiny_model[0], [(64, [(20, 1), (30, 2)]), (32, [(5, 1)])], 4, 2, 128, 16, seed=9)
        ints = s.c.ints
        table = s.c.book.table()
        table[0, 1] = 10 ** 6
        for over, code in ((dict(seqs=ints([0, 9, 2])), 1), (dict(seqs=ints([-1, 1, 2])), 1), (dict(cu_rows=ints([0, 3, 2, 4])), 5),
                           (dict(cu_rows=ints([0, 1, 3, 9])), 5), (dict(max_len=80), 5), (dict(max_rows=1), 5), (dict(max_shared=32), 5),
                           (dict(max_own=8), 5), (dict(max_group_rows=2), 5), (dict(cu_groups=ints([0, 2, 7])), 5), (dict(cu_groups=ints([1, 2, 3])), 5),
                           (dict(shared=ints([84, 32])), 5), ("table", 1)):
            if over == "table":
                dev.put(table, s.c.at["table"])
                over = {}
            if over.get("max_len") == 80:
                over.update(max_shared=64, max_own=80)
            for planned in ({}, dict(max_len=1040)):
                if "max_len" in over and planned:
                    continue
                with pytest.raises(Q3Error):
                    s.run(s.batch(**over, **planned))
                st = dev.stream()
                s.run(s.batch(**over, **planned), stream=st)
                assert s.c.c.status(stream=st)[0] == code, (over, planned)
        s.c.put()
        s.check(*s.run(s.batch()))
        b = s.batch(max_rows=0)
        with pytest.raises(Q3Error, match="max_rows"):
            s.run(b)


def test_attention_on_two_streams_and_in_a_graph(tiny_model):
    with Device() as dev:
        steps = [Step(dev, tiny_model[0], GROUPS[g], 4, 2, 128, 16, seed=20 + g) for g in (3, 4)]
        jobs = []
        for s in steps:
            b = s.batch()
            n = s.c.c.attention_workspace_bytes(b, s.heads)
            jobs.append((s, b, dev.put(s.q), dev.raw(s.q.nbytes), (dev.raw(n), n), s.run(b)[0], dev.stream()))
        for _ in range(3):
            for s, b, q, o, ws, want, st in jobs:
                s.c.c.attention(s.layer, q, o, b, s.heads, workspace=ws, stream=st)
            for s, b, q, o, ws, want, st in jobs:
                dev.wait(st)
                assert np.array_equal(dev.get(o, want.shape, np.uint16), want)
        st = jobs[0][-1]
        graph = dev.capture(st, lambda: [s.c.c.attention(s.layer, q, o, b, s.heads, workspace=ws, stream=st) for s, b, q, o, ws, _, _ in jobs])
        for rep in range(4):
            for s, b, q, o, ws, want, _ in jobs:
                dev.put(np.zeros_like(want), o)
            assert dev.h.hipGraphLaunch(graph, st) == 0
            dev.wait(st)
            for s, b, q, o, ws, want, _ in jobs:
                assert np.array_equal(dev.get(o, want.shape, np.uint16), want), rep
                s.check(*s.run(b))       # eager work between the replays
        dev.h.hipGraphExecDestroy(graph)


def test_decode_steps_of_several_hypotheses(tiny_model):
    """What a beam search does for one layer, step by step: the hypotheses of two clips leave their prompts, are reordered by
    parents, get room, project q / k / v on 8-bit weights, write their rows, attend with the prompt read once, project the result.
    Every stage is checked on the device's own input of that stage, so that no rounding of an earlier one excuses a later one."""
    from q3asr import AttentionBatch, Int8Linear, quantize_rows
    from test_gpu_serving_i8 import _quantize64
    rng = np.random.default_rng(77)
    model, hidden, heads, kv, d, hyps, clips = tiny_model[0], 256, 4, 2, 128, 3, 2
    qkv, n = (heads + 2 * kv) * d, hyps * clips
    with Device() as dev:
        def weights(rows, cols):
            w = bf16_bits(rng.standard_normal((rows, cols)) / np.sqrt(cols))
            q, s = dev.raw(rows * cols), dev.raw(4 * rows)
            quantize_rows(model, dev.put(w), rows, cols, q, s)
            ref = _quantize64(bf16_vals(w))
            return Int8Linear(model, q, s, rows, cols), ref

        w_qkv, w_o = weights(qkv, hidden), weights(hidden, heads * d)

        def linear(lin, ref, x_bits, rows, x, o):
            ws = lin.workspace_bytes(rows)
            lin(x, rows, o, workspace=(dev.raw(ws), ws))
            got = bf16_vals(dev.get(o, (rows, lin.N), np.uint16)).astype(np.float64)
            s, q = _quantize64(bf16_vals(x_bits))
            want = (q @ ref[1].T).astype(np.float64) * s.astype(np.float64)[:, None] * ref[0].astype(np.float64)
            assert (np.abs(got - want) <= 2.0 ** -8 * 1.01 * np.abs(want) + 1e-30).all()

        prompts = [37, 50]
        c = Cache(dev, model, seqs=clips + n, width=8, pages=80, layers=1, heads=kv, dim=d, pg=16, seed=3)
        c.reserve([0, 1], prompts)
        seqs = list(range(clips, clips + n))
        c.fork(seqs, [i // hyps for i in range(n)])
        cu_groups, shared = c.ints([0, hyps, n]), c.ints([p // 16 * 16 for p in prompts])
        for step in range(6):
            if step:
                parents = [clips + g * hyps + int(p) for g in range(clips) for p in rng.integers(0, hyps, hyps)]
                c.fork(seqs, parents)
            c.reserve(seqs, [1] * n)
            x = bf16_bits(rng.standard_normal((n, hidden)))
            proj = dev.raw(2 * n * qkv)
            linear(*w_qkv, x, n, dev.put(x), proj)
            rows = dev.get(proj, (n, qkv), np.uint16)
            b = AttentionBatch(seqs=c.ints(seqs), cu_rows=c.ints(range(n + 1)), n=n, rows=n, n_groups=clips, cu_groups=cu_groups, shared=shared,
                               max_rows=1, max_group_rows=hyps, max_len=max(c.book.lens), max_shared=48, max_own=16 + step + 1)
            c.c.write(0, proj + 2 * heads * d, proj + 2 * (heads + kv) * d, b, k_ld=qkv, v_ld=qkv)
            c.book.write(0, rows[:, heads * d:(heads + kv) * d], rows[:, (heads + kv) * d:], seqs, list(range(n + 1)))
            c.check()
            o, nb = dev.raw(2 * n * heads * d), c.c.attention_workspace_bytes(b, heads)
            c.c.attention(0, proj, o, b, heads, q_ld=qkv, workspace=(dev.raw(nb), nb))
            att = dev.get(o, (n, heads * d), np.uint16)
            for i, sq in enumerate(seqs):
                k, v = c.book.keys(0, sq)
                q = bf16_vals(rows[i, :heads * d]).astype(np.float64).reshape(1, heads, d)
                want, _, size, slack = attention64(q, k, v, c.book.lens[sq], 1, heads, d ** -0.5)
                got = bf16_vals(att[i]).astype(np.float64).reshape(want.shape)
                assert (np.abs(got - want) <= attention_bounds(want, size, slack, c.book.lens[sq])).all(), (step, i)
            linear(*w_o, att, n, o, dev.raw(2 * n * hidden))
        c.free(seqs)
        c.compact()
        c.check()
