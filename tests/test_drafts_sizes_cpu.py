"""What the draft operators keep on the host between calls."""


def test_what_is_kept_of_sizes_is_bounded():
    """A server meets any number of requests a step: the sizes of a call's scratch are not remembered without end."""
    from tinyinfer_b200 import ops
    before = len(ops._scratch_floats)
    words = {ops._verify_scratch_words(s, d, 32000, True, False) for s in range(1, 3001) for d in (1, 4)}
    assert len(words) > 3000 and len(ops._scratch_floats) == before
    assert ops._verify_scratch_words.cache_info().currsize <= 4096
    # rows of tiles of 256 words, then 8 words a row
    assert ops._verify_scratch_words(2, 3, 32000, True, False) == 2 * 4 * (4 * 256 + 8)
