"""Which entry of a batch an attention's error names."""
import pytest

from serving_kit import Device
from test_gpu_serving_attention import Step

pytestmark = pytest.mark.gpu

BAD_INDEX, BAD_BATCH = 1, 5


def _reversed(s):
    """The batch's lists from the last group and sequence to the first, so that an entry's number is not its sequence's."""
    n = len(s.seqs)
    s.seqs, s.shared, s.lens = s.seqs[::-1], s.shared[::-1], s.lens[::-1]
    s.cu_groups = [n - x for x in s.cu_groups[::-1]]


def _status(dev, s, batch):
    st = dev.stream()
    s.run(batch, stream=st)
    return s.c.c.status(stream=st)[:2]


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("groups", [3, 400])
def test_a_wrong_page_names_its_entry(tiny_model, groups, dim):
    """A page number out of range in a sequence's own pages, and in its group's shared ones, which the group's first sequence stands for;
    in one launch, through the plan in every workgroup (3 groups) or in a launch of its own (400), and without groups."""
    with Device() as dev:
        s = Step(dev, tiny_model[0], [(40, [(9, 1), (30, 1), (5, 1)])] * groups, 4, 2, dim, 16, seed=3)
        _reversed(s)
        right = s.c.book.table()
        for entry, slot in ((3, 4), (7, 2), (8, 4), (0, 0), (3, 1), (6, 0), (3 * groups - 3, 1)):
            table = right.copy()
            seq = s.seqs[entry]
            if slot * 16 >= s.lens[entry]:
                slot = (s.lens[entry] - 1) // 16
            table[seq, slot] = (10 ** 6, -1)[entry % 2]
            dev.put(table, s.c.at["table"])
            for over in ({}, dict(max_len=1040), dict(grouped=False), dict(grouped=False, max_len=1040)):
                assert _status(dev, s, s.batch(**over)) == (BAD_INDEX, entry), (entry, slot, over)
        s.c.put()
        for over in ({}, dict(max_len=1040)):
            assert _status(dev, s, s.batch(**over)) == (0, 0)


def test_wrong_bounds_name_their_entry(tiny_model):
    with Device() as dev:
        s = Step(dev, tiny_model[0], [(64, [(20, 1), (30, 1), (7, 1)]), (32, [(5, 1), (90, 1)])], 4, 2, 128, 16, seed=9)
        _reversed(s)
        ints = s.c.ints
        for over, want in ((dict(seqs=ints([4, 3, 2, 9, 0])), (BAD_INDEX, 3)), (dict(seqs=ints([4, 3, -1, 1, 0])), (BAD_INDEX, 2)),
                           (dict(cu_groups=ints([0, 2, 7])), (BAD_BATCH, 2)), (dict(cu_groups=ints([1, 2, 5])), (BAD_BATCH, 0)),
                           (dict(cu_groups=ints([0, 2, 4])), (BAD_BATCH, 4)), (dict(max_own=80), (BAD_BATCH, 0)),
                           (dict(max_shared=48), (BAD_BATCH, 2))):
            for form in ({}, dict(max_len=1040)):
                assert _status(dev, s, s.batch(**over, **form)) == want, (over, want, form)
