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


def test_misaligned_numbers_are_refused(lib, handle):
    """Scales, biases and lists are read four bytes at a time, into LDS too, where the low bits of an address would be dropped."""
    P = 1 << 20

    def refused(rc):
        return rc != 0 and "misaligned" in lib.q3asr_last_error().decode()

    def linear(sw=P, bias=P):
        return lib.q3asr_i8_linear(handle, P, 1, 64, P, 64, sw, bias, 4, 8, 64, P, 1, 8, P, 1 << 20, None)

    def matmul(sa=P, sw=P, bias=P):
        return lib.q3asr_i8_matmul(handle, P, 64, sa, P, 64, sw, bias, 4, 8, 64, P, 1, 8, None)

    for rc in (linear(sw=P + 2), linear(bias=P + 1), matmul(sa=P + 2), matmul(sw=P + 3), matmul(bias=P + 2),
               lib.q3asr_i8_quantize(handle, P, 0, 20, 3, 20, P, 32, P + 2, None)):
        assert refused(rc)
    c = ctypes.byref(q3lib.Q3Pages(k=P, v=P, table=P, lens=P, refs=P, status=P, layers=1, pages=10, kv_heads=2, head_dim=128, page_tokens=16, max_seqs=4,
                                   max_seq_pages=5, workspace=P, workspace_bytes=1 << 20))
    for args in ((P + 1, P), (P, P + 2)):
        assert refused(lib.q3asr_pages_fork(handle, c, *args, 1, None))
        assert refused(lib.q3asr_pages_reserve(handle, c, *args, 1, None))
    assert refused(lib.q3asr_pages_free(handle, c, P + 2, 1, None))
    base = dict(seqs=P, cu_rows=P, cu_groups=P, shared=P, n=4, rows=6, n_groups=2, max_rows=2, max_group_rows=4, max_len=70, max_shared=32, max_own=40)
    for name in ("seqs", "cu_rows", "cu_groups", "shared"):
        b = ctypes.byref(q3lib.AttentionBatch(**{**base, name: P + 2}))
        assert refused(lib.q3asr_pages_write(handle, c, 0, P, 256, P, 256, b, None)), name
        assert refused(lib.q3asr_paged_attention(handle, c, 0, P, 512, 4, 0.1, b, P, 512, P, P, 1 << 30, None)), name
