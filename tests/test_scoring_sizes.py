"""What score_tokens asks for and refuses by its sizes alone, on the CPU."""

from whisper_trt_b200 import _lib


def test_scratch_is_bounded():
    """Whatever the rows: the scratch holds a pass of them, not the logits' size again."""
    size = _lib.load().wt_score_tokens_workspace
    for rows in (1, 160, 7136, 30000, 2**24):
        for top in (0, 1, 5, 16):
            for vocab in (1000, 51866, 2**20):
                assert size(rows, vocab, 1280, top) <= 330 * 2**20, (rows, vocab, top)
    assert size(7136, 51866, 1280, 5) >= 7136 * 4 * (4 + 12 + 5 * 32)


def test_unsupported_sizes_need_no_scratch():
    """What the call refuses has no scratch (its size would have passed the counters)."""
    size = _lib.load().wt_score_tokens_workspace
    for rows, vocab in ((2**24 + 1, 51866), (4, 2**20 + 1), (2**31 - 1, 2**31 - 1), (4, 2**31 - 1), (2**31 - 1, 4)):
        assert size(rows, vocab, 64, 5) == 0, (rows, vocab)
    assert size(2**24, 2**20, 64, 5) > 0
