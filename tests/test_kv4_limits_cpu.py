"""Limits of the 4-bit cache's calls, without a GPU."""
from nanoquantization_b200 import _lib

P = 1 << 20        # an address that is aligned and never reached


def test_sums_of_tiles_stay_within_31_bits():
    """A call's tiles are numbered in 32 bits, over sequences whose numbers on the device are not known to be the host's."""
    lib, cache = _lib.load(), _lib.Kv4(P, P, 4, 2, 16)
    call = lambda tiles: lib.nqb200_kv4_prompt_attention(P, 512, cache, P, 8, P, P, P, 1, 4, 4, 100, tiles, 4, 0.1, 0, None, 0, None, None)  # noqa: E731
    for tiles in ((1 << 24) + 1, (2**31 - 1) // 2):
        assert call(tiles) == 1 and lib.nqb200_kv4_prompt_scratch_bytes(1, 4096, 4096, 1 << 20, tiles, 32, 2) == 0
    assert lib.nqb200_kv4_prompt_scratch_bytes(1, 4096, 4096, 1 << 20, 1 << 24, 32, 2) >= 2 << 40
