"""The paged KV cache's table operations against a book kept in Python lists: tables, lengths, counts and contents, bit for bit."""
import numpy as np
import pytest

from conftest import bf16_bits
from q3asr.lib import Q3Error
from serving_kit import Cache, Device

pytestmark = pytest.mark.gpu


def _filled(dev, model, lens, **kw):
    """A cache whose first sequences have these lengths."""
    c = Cache(dev, model, **kw)
    c.reserve(list(range(len(lens))), lens)
    return c


@pytest.mark.parametrize("pg", [16, 32, 256])
@pytest.mark.parametrize("dim", [64, 128])
def test_fork_and_reserve_copy_on_write(tiny_model, pg, dim):
    with Device() as dev:
        c = _filled(dev, tiny_model[0], [0, 1, pg - 1, pg, pg + 1, 5 * pg + 3], seqs=20, width=8, pages=90, layers=3, heads=3, dim=dim, pg=pg)
        c.check()
        c.fork([6, 7, 8, 9, 10, 11], [5, 5, 2, 3, 0, 1])
        c.check()
        c.reserve([6, 7, 8, 9, 10, 11], [1, pg, 2, 1, 3, 0])     # 5 keeps its page, its heirs copy
        c.check()
        c.reserve([5, 4, 3, 2, 1, 0], [1, 1, 1, 1, 1, 1])
        c.check()
        # all holders of one page in the list: the first of them keeps it
        c.fork([12, 13, 14], [4, 4, 4])
        c.reserve([13, 4, 14, 12], [1, 2, 3, 4])
        c.check()
        # one of them adds nothing: it holds on to the page, so the others copy
        c.fork([15, 16], [13, 13])
        c.reserve([16, 13, 15], [1, 0, 1])
        c.check()
        c.free([0, 5, 6, 7, 9])
        c.check()
        assert c.compact() == sum(r > 0 for r in c.book.refs)
        c.check()
        assert c.c.status()[:3] == (0, 0, 0)


def test_beam_reordering_reads_the_table_before_it_writes(tiny_model):
    rng = np.random.default_rng(3)
    with Device() as dev:
        c = _filled(dev, tiny_model[0], [30, 31, 45, 64, 7, 16, 1, 100], seqs=8, width=16, pages=300, layers=2)
        for step in range(12):
            parents = rng.integers(0, 8, 8).tolist()
            c.fork(list(range(8)), parents)
            order = rng.permutation(8).tolist()
            c.reserve(order, rng.integers(0, 6, 8).tolist())
            c.check()
        c.fork([0, 1], [1, 0])               # a swap
        c.check()
        c.fork([3], [3])                     # a sequence onto itself
        c.check()
        c.fork([2, 4], [-1, 2])              # gives up what the other takes over
        c.check()
        c.compact()
        c.check()


@pytest.mark.parametrize("n,width", [(3, 2), (1500, 3), (40, 700), (2100, 2)])
def test_lists_of_any_length(tiny_model, n, width):
    """More entries than threads; longer tables than threads; many pages."""
    rng = np.random.default_rng(n)
    with Device() as dev:
        c = Cache(dev, tiny_model[0], seqs=2 * n, width=width, pages=2 * n * width + 5, layers=1, heads=1, dim=64, seed=1)
        c.reserve(rng.permutation(n).tolist(), rng.integers(0, 16 * width - 20, n).tolist())
        c.check()
        c.fork((n + rng.permutation(n)).tolist(), rng.integers(-1, n, n).tolist())
        c.check()
        c.reserve(rng.permutation(2 * n).tolist(), rng.integers(0, 17, 2 * n).tolist())
        c.check()
        c.free(rng.permutation(2 * n)[:n].tolist())
        c.check()
        c.compact()
        c.check()
        c.reserve([0], [1])
        c.check()


def test_compact_of_full_and_empty_pools(tiny_model):
    with Device() as dev:
        c = Cache(dev, tiny_model[0], seqs=4, width=64, pages=128, layers=2, heads=2, dim=64)
        assert c.compact() == 0
        c.check()
        c.reserve([0, 1, 2, 3], [512, 512, 512, 512])
        c.check()
        assert c.compact() == 128           # nothing to move
        c.check()
        c.free([0, 2])
        assert c.compact() == 64
        c.check()
        assert c.compact() == 64
        c.check()
        assert c.c.status()[3] == 64
        c.c.reset()
        assert c.state()[1].tolist() == [0] * 4 and (c.state()[0] == -1).all() and (c.state()[2] == 0).all()


def test_refused_calls_change_nothing(tiny_model):
    """Wrong entries anywhere in the list: nothing of the call is done, the error names the entry, the cache stays usable."""
    with Device() as dev:
        c = _filled(dev, tiny_model[0], [20, 40, 8], seqs=6, width=4, pages=12)
        cases = [(lambda s: c.c.fork(c.ints([3, 6]), c.ints([0, 0]), 2, s), "out of range.*entry 1", 1),
                 (lambda s: c.c.fork(c.ints([3, -2]), c.ints([0, 0]), 2, s), "out of range.*entry 1", 1),
                 (lambda s: c.c.fork(c.ints([3, 4]), c.ints([0, 9]), 2, s), "out of range.*entry 1", 1),
                 (lambda s: c.c.fork(c.ints([3, 4]), c.ints([-2, 0]), 2, s), "out of range.*entry 0", 1),
                 (lambda s: c.c.fork(c.ints([3, 4, 3]), c.ints([0, 1, 2]), 3, s), "named twice", 2),
                 (lambda s: c.c.free(c.ints([1, 1]), 2, s), "named twice", 2),
                 (lambda s: c.c.reserve(c.ints([0, 1, 0]), c.ints([1, 1, 1]), 3, s), "named twice", 2),
                 (lambda s: c.c.reserve(c.ints([0, 7]), c.ints([1, 1]), 2, s), "out of range.*entry 1", 1),
                 (lambda s: c.c.reserve(c.ints([0, -2]), c.ints([1, 1]), 2, s), "out of range.*entry 1", 1),
                 (lambda s: c.c.reserve(c.ints([0, 1]), c.ints([1, -1]), 2, s), "out of range.*entry 1", 1),
                 (lambda s: c.c.reserve(c.ints([0, 1]), c.ints([1, 25]), 2, s), "outgrow.*entry 1", 4),
                 (lambda s: c.c.reserve(c.ints([3, 4]), c.ints([64, 2 ** 31 - 1]), 2, s), "outgrow.*entry 1", 4),
                 (lambda s: c.c.reserve(c.ints([3, 4]), c.ints([64, 16]), 2, s), None, 0)]
        for call, text, code in cases[:-1]:
            with pytest.raises(Q3Error, match=text):
                call(None)
            c.check()
        # 6 pages are free: one too few
        c.reserve([3], [48])
        with pytest.raises(Q3Error, match="not enough free pages .1 short"):
            c.c.reserve(c.ints([4]), c.ints([64]), 1)
        c.check()
        # without waiting: the first error is kept until it is asked for, later good calls are done
        s = dev.stream()
        for call, text, code in cases[:-1]:
            call(s)
            c.c.free(c.ints([9]), 1, s)
            c.c.fork(c.ints([5]), c.ints([5]), 1, s)
            assert c.c.status(stream=s)[0] == code
            assert c.c.status(stream=s)[0] == 0
            c.check()
        with pytest.raises(Q3Error, match="more entries than sequences"):
            c.c.fork(c.ints(range(7)), c.ints(range(7)), 7)
        c.c.fork(0, 0, 0)                    # nothing to do
        c.check()


@pytest.mark.parametrize("seqs,width", [(600, 1), (600, 9), (4096, 2), (5000, 1), (5000, 3)])
def test_the_first_repeated_entry_is_named(tiny_model, seqs, width):
    """Few and many sequences, short and long tables: the entry that is reported is the first one that names a sequence again."""
    rng = np.random.default_rng(seqs + width)
    with Device() as dev:
        c = _filled(dev, tiny_model[0], [3, 16, 9], seqs=seqs, width=width, pages=30)
        for n, later in ((600, (599,)), (600, (3, 400)), (40, (17, 18, 39)), (seqs, (seqs - 1, seqs // 2))):
            names = rng.permutation(seqs)[:n]
            for at in later:
                names[at] = names[rng.integers(0, min(later))]
            first = min(later)
            zeros = c.ints(np.zeros(n))
            for call in (lambda: c.c.fork(c.ints(names), zeros, n), lambda: c.c.free(c.ints(names), n), lambda: c.c.reserve(c.ints(names), zeros, n)):
                with pytest.raises(Q3Error, match=f"named twice .entry {first}."):
                    call()
        c.check()
        order = rng.permutation(seqs).tolist()          # the whole cache in one call
        c.fork(order, [2 if q == 2 else -1 if q % 2 else 0 for q in order])
        c.check()


@pytest.mark.parametrize("n", [6, 700])
def test_entries_of_minus_one_stand_for_none(tiny_model, n):
    """Lists of fixed length: -1 is skipped in fork, free and reserve, however often it stands there."""
    with Device() as dev:
        c = _filled(dev, tiny_model[0], [20, 37, 5], seqs=max(n, 8), width=6, pages=60, layers=2)
        pad = [-1] * (n - 4)
        c.c.fork(c.ints([3, -1, 4, 5] + pad), c.ints([0, 2, 1, -1] + [1] * len(pad)), n)
        c.book.fork([3, 4, 5], [0, 1, -1])
        c.check()
        c.c.reserve(c.ints([-1, 4, 3, -1] + pad), c.ints([9, 1, 20, 0] + [7] * len(pad)), n)
        c.book.reserve([4, 3], [1, 20])
        c.check()
        c.c.free(c.ints([-1, -1, 1, 4] + pad), n)
        c.book.fork([1, 4], [-1, -1])
        c.check()


def test_write_puts_rows_at_the_ends(tiny_model):
    from q3asr import AttentionBatch
    rng = np.random.default_rng(8)
    with Device() as dev:
        c = _filled(dev, tiny_model[0], [20, 5, 33, 16, 1, 70], seqs=8, width=6, pages=30, layers=3, heads=3, dim=64, pg=16)
        seqs, cu = [5, 0, 4, 2, 1], [0, 18, 18, 19, 22, 27]      # sequence 0 has no row, 1 nothing but rows
        ld = 3 * 64 + 8
        k, v = (bf16_bits(rng.standard_normal((27, ld))) for _ in range(2))
        b = AttentionBatch(seqs=c.ints(seqs), cu_rows=c.ints(cu), n=5, rows=27, max_rows=18, max_len=96)
        c.c.write(1, dev.put(k), dev.put(v), b, k_ld=ld, v_ld=ld)
        c.book.write(1, k[:, :192], v[:, :192], seqs, cu)
        c.check()
        # rows behind the last sequence's are left out
        b = AttentionBatch(seqs=c.ints(seqs), cu_rows=c.ints(cu), n=5, rows=40, max_rows=18, max_len=96)
        k2 = bf16_bits(rng.standard_normal((40, ld)))
        c.c.write(0, dev.put(k2), dev.put(k2), b, k_ld=ld, v_ld=ld)
        c.book.write(0, k2[:, :192], k2[:, :192], seqs, cu)
        c.check()
        # a shared page is not written, a sequence named twice keeps its first row, rows before a sequence's start are left out
        c.fork([6], [2])
        at = dev.put(k)
        for seqs, cu, code in (([6, 0], [0, 1, 2], 5), ([0, 1, 0], [0, 1, 2, 3], 2), ([9, 0], [0, 1, 2], 1), ([4, 0], [0, 2, 3], 5)):
            b = AttentionBatch(seqs=c.ints(seqs), cu_rows=c.ints(cu), n=len(seqs), rows=cu[-1], max_rows=2, max_len=96)
            s = dev.stream()
            c.c.write(2, at, at, b, k_ld=ld, v_ld=ld, stream=s)
            assert c.c.status(stream=s)[0] == code
            if seqs == [6, 0]:
                c.book.write(2, k[1:2, :192], k[1:2, :192], [0], [0, 1])
            elif seqs == [0, 1, 0]:
                c.book.write(2, k[:2, :192], k[:2, :192], [0, 1], [0, 1, 2])
            elif seqs == [9, 0]:
                c.book.write(2, k[1:2, :192], k[1:2, :192], [0], [0, 1])
            else:
                c.book.write(2, k[1:3, :192], k[1:3, :192], [4, 0], [0, 1, 2])
            c.check()


def test_page_calls_in_a_graph(tiny_model):
    """fork, reserve, free and compact captured once and replayed: every replay does what the eager calls do."""
    with Device() as dev:
        c = _filled(dev, tiny_model[0], [37, 50, 5], seqs=10, width=8, pages=64, layers=2)
        dst, src, add, gone = [3, 4, 5, 6], [0, 0, 1, 2], [1, 2, 15, 40], [4, 6]
        d = [c.ints(x) for x in (dst, src, add, gone)]
        s = dev.stream()

        def calls():
            c.c.fork(d[0], d[1], 4, s)
            c.c.reserve(d[0], d[2], 4, s)
            c.c.free(d[3], 2, s)
            c.c.compact(s)

        graph = dev.capture(s, calls)
        for rep in range(4):
            assert dev.h.hipGraphLaunch(graph, s) == 0
            dev.wait(s)
            c.book.fork(dst, src)
            c.book.reserve(dst, add)
            c.book.fork(gone, [-1, -1])
            c.book.compact()
            c.check()
            c.reserve([0, 7], [1, rep])          # eager calls between the replays
            c.check()
        dev.h.hipGraphExecDestroy(graph)
