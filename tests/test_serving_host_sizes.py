"""Sizes and addresses that the serving operators refuse, beside those of test_serving_host; no GPU needed."""
import ctypes

import pytest

from q3asr import lib as q3lib


@pytest.fixture(scope="module")
def lib():
    return q3lib.load()


@pytest.fixture()
def handle():
    """Stands for a model: a call that is refused never looks into it."""
    held = ctypes.create_string_buffer(1 << 14)
    yield ctypes.addressof(held)


def test_workspace_sizes_are_refused_like_the_calls(lib, handle):
    """A size that the product refuses has no workspace either."""
    big = 2 ** 24
    assert lib.q3asr_i8_workspace(handle, big, 8, 64) == -1 and lib.q3asr_i8_workspace(handle, 8, big, 64) == -1
    assert lib.q3asr_i8_workspace(handle, big - 1, 8, 64) >= (big - 1) * 68
    from q3asr import Int8Linear, PagedKVCache

    class Model:
        _lib, _h = lib, handle

    with pytest.raises(ValueError, match="out of range"):
        Int8Linear(Model, 1 << 20, 1 << 20, 8, 64).workspace_bytes(big)
    P = 1 << 20
    c = PagedKVCache(Model, k=P, v=P, layers=1, pages=0, kv_heads=1, head_dim=64, page_tokens=16, table=P, lens=P, refs=P, status=P, max_seqs=1, max_seq_pages=1)
    with pytest.raises(ValueError, match="out of range"):
        c.workspace_bytes()
