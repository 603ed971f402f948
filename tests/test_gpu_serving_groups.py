"""Groups of the attention's batch whose entries partly stand for no sequence: hypotheses that have ended in lists of fixed length."""
import numpy as np
import pytest

from q3asr.lib import Q3Error
from serving_kit import Device
from test_gpu_serving_attention import Step

pytestmark = pytest.mark.gpu

BAD_BATCH = 5


def _end(s, places):
    """The sequences at these places of the list become -1 entries without rows."""
    keep = [r for i in range(len(s.seqs)) if i not in places for r in range(s.cu[i], s.cu[i + 1])]
    s.q = s.q[keep]
    for i in places:
        s.seqs[i], s.rows[i] = -1, 0
    s.cu = np.concatenate([[0], np.cumsum(s.rows)]).tolist()


def _own(s):
    """The most tokens that a sequence in the list has behind its group's whole shared pages."""
    pg = s.c.book.pg
    return max(s.lens[i] - n // pg * pg for n, a, b in zip(s.shared, s.cu_groups, s.cu_groups[1:]) for i in range(a, b) if s.seqs[i] >= 0)


GROUPS = [(405, [(30, 1), (3, 1), (41, 2), (1, 1), (17, 1)]), (70, [(9, 1), (2, 1), (40, 1)]), (5, [(50, 1), (1, 1)])]
ENDED = [(0,), (2,), (4,), (0, 1), (0, 4, 5), (5, 6), (0, 1, 2, 3, 4), (0, 2, 5, 7, 8), (8,)]


@pytest.mark.parametrize("heads,kv,dim", [(4, 2, 128), (14, 7, 64)])
@pytest.mark.parametrize("ended", ENDED)
def test_ended_hypotheses_leave_their_group_alone(tiny_model, ended, heads, kv, dim):
    """-1 at the first, a middle and the last place of a group, and a group of nothing else, under the tightest bounds: the others read
    all of their keys, in one launch, through the plan, and without groups."""
    with Device() as dev:
        s = Step(dev, tiny_model[0], GROUPS, heads, kv, dim, 16, seed=sum(ended))
        _end(s, ended)
        for b in (s.batch(max_own=_own(s)), s.batch(max_own=_own(s), max_len=1040), s.batch(grouped=False), s.batch(grouped=False, max_len=1040)):
            s.check(*s.run(b))
            assert s.c.c.status()[:3] == (0, 0, 0)


@pytest.mark.parametrize("place", [(0,), (1,), (2,), (0, 1)])
def test_ended_hypotheses_in_a_batch_that_a_launch_plans(tiny_model, place):
    """The same over 1024 groups and sequences."""
    with Device() as dev:
        s = Step(dev, tiny_model[0], [(40, [(3, 1), (5, 2), (2, 1)])] * 300, 4, 2, 64, 16, seed=7)
        _end(s, [3 * g + i for g in range(0, 300, 2) for i in place])
        s.check(*s.run(s.batch(max_own=_own(s), max_len=1040)))
        assert s.c.c.status()[:3] == (0, 0, 0)


@pytest.mark.parametrize("ended", [1, 7, 8, 9, 63, 64, 65, 129])
def test_many_ended_hypotheses_in_front(tiny_model, ended):
    """Any number of -1 entries before a group's first sequence, in a group of its own size and beside another."""
    with Device() as dev:
        s = Step(dev, tiny_model[0], [(50, [(4, 1)] * 2), (90, [(1 + i % 7, 1) for i in range(ended + 2)])], 4, 2, 128, 16, seed=ended)
        _end(s, range(2, 2 + ended))
        s.check(*s.run(s.batch(max_own=_own(s), max_len=1040)))
        assert s.c.c.status()[:3] == (0, 0, 0)


def test_a_bound_that_an_ended_hypothesis_hides_is_reported(tiny_model):
    """max_own one token short: an error whether or not the group begins with -1, never fewer keys in silence."""
    with Device() as dev:
        for ended in ((), (0,), (0, 1), (4,)):
            s = Step(dev, tiny_model[0], GROUPS[:1], 4, 2, 128, 16, seed=11)
            _end(s, ended)
            for over in ({}, dict(max_len=1040)):
                with pytest.raises(Q3Error, match="bounds"):
                    s.run(s.batch(max_own=_own(s) - 1, **over))
                st = dev.stream()
                s.run(s.batch(max_own=_own(s) - 1, **over), stream=st)
                assert s.c.c.status(stream=st)[0] == BAD_BATCH, (ended, over)
                s.check(*s.run(s.batch(max_own=_own(s), **over)))
