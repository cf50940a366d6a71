"""What nvk_fp4_attention_workspace_size takes, on the CPU (0: not supported)."""
import pytest

from nanovllm_amd import _lib


def size(batch=4, max_q=1, max_k=0, hq=16, hkv=8, d=128, bs=256, blocks=16):
    return _lib.load().nvk_fp4_attention_workspace_size(batch, max_q, max_k, hq, hkv, d, bs, blocks)


@pytest.mark.parametrize("sizes", [{}, {"d": 64}, {"bs": 16}, {"bs": 48}, {"hq": 8}, {"hq": 128},
                                   {"batch": 2048}, {"max_q": 65}, {"max_q": 4096, "max_k": 4096},
                                   {"hq": 24, "max_q": 100}, {"batch": 1, "blocks": 4096}])
def test_supported(sizes):
    assert size(**sizes) > 0


@pytest.mark.parametrize("sizes", [{"batch": 0}, {"batch": 2049}, {"max_q": 0}, {"d": 96}, {"bs": 8},
                                   {"bs": 100}, {"hq": 12}, {"hq": 136}, {"blocks": 0},
                                   {"blocks": 1 << 23}, {"batch": -1}, {"hkv": 0}, {"hq": 0},
                                   {"max_q": (1 << 31) - 1}])
def test_not_supported(sizes):
    assert size(**sizes) == 0


def test_long_queries_of_many_sequences():
    """Through pages the (tile, chunk) pairs of the direct kernel are not counted: 512 sequences with
    up to 16384 queries over 40960 keys would be 2.7e9 of them.  The pages stay within 512 MiB."""
    n = size(batch=512, max_q=16384, max_k=40960, blocks=160)
    assert 0 < n < 1 << 30
    assert size(batch=512, max_q=16384, d=64, blocks=160) == 0


def test_pages_follow_the_bound_on_the_keys():
    wide = size(batch=2, max_q=500, blocks=64)
    assert size(batch=2, max_q=500, max_k=1000, blocks=64) < wide
    assert size(batch=2, max_q=500, max_k=1 << 30, blocks=64) == wide
