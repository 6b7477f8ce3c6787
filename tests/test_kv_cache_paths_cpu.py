"""Which path attention over the 8-bit cache takes, and what memory that may need (no GPU)."""
import pytest

from transformerengine_b200.attention import kv_cache as kc


@pytest.mark.parametrize("n,hq,hk,max_q,expands", [
    (8, 32, 8, 32, False), (8, 32, 8, 64, True), (8, 32, 8, 128, True), (1, 32, 8, 128, False), (64, 32, 8, 64, True),
    (2, 32, 8, 1024, True), (64, 32, 8, 1, False), (256, 64, 8, 4, False), (1, 8, 8, 64, False)])
def test_sequences_alike(n, hq, hk, max_q, expands):
    assert kc._expands(n, hq, hk, 128, max_q, n * max_q, 8000) == expands


@pytest.mark.parametrize("chunks,singles,expands", [(1, 63, False), (8, 56, True), (8, 8, True), (1, 1, True), (1, 255, False)])
def test_chunks_beside_single_tokens(chunks, singles, expands):
    assert kc._expands(chunks + singles, 32, 8, 128, 1024, 1024 * chunks + singles, 8000) == expands


def test_no_expansion_beyond_its_memory():
    for hk, d in ((8, 128), (1, 128), (64, 128)):
        most = kc._EXPAND_BYTES // (4 * hk * d)
        for max_kv in (most // 2, most + 1000, 2 ** 31 - 1):
            fits = kc._expansion_bytes(64, hk, d, 1024, max_kv) <= kc._EXPAND_BYTES
            assert fits == (max_kv < most)
            assert kc._expands(4, 64, hk, d, 1024, 4096, max_kv) <= fits
    # keys and values in 16 bits over whole 128-token blocks, a 32-bit number per query row
    assert kc._expansion_bytes(8, 2, 128, 1, 129) == 2 * 2 * 256 * 2 * 128 + 8 * 128 * 4
