"""The lines between prefixes that are read once and those that each sequence reads by itself, on both sides of what was measured (no GPU)."""

import pytest

from kernel_rush_kawk_b200.cache.prefix import longer_steps_share, single_tokens_share


@pytest.mark.parametrize("n,length,shares", [(2, 4096, False), (2, 8192, True), (4, 2048, False), (4, 4096, True), (16, 1024, False), (16, 2048, True), (64, 256, False),
                                             (64, 1024, True)])
def test_single_tokens(n, length, shares):
    assert single_tokens_share([n], [length], 4096) is shares


@pytest.mark.parametrize("n,tokens,length,shares", [
    (2, 4, 512, False), (2, 4, 1024, True), (4, 4, 1024, False), (4, 4, 2048, True), (4, 16, 1024, False), (4, 16, 2048, True), (8, 2, 512, False), (8, 2, 1024, True),
    (8, 8, 1024, False), (8, 8, 2048, True), (8, 30, 512, False), (8, 30, 1024, True), (32, 8, 512, True), (16, 31, 512, True), (4, 60, 1024, False), (4, 60, 4096, True),
    (16, 60, 4096, False), (2, 250, 1024, False), (2, 250, 4096, True), (4, 250, 4096, False)])
def test_longer_steps(n, tokens, length, shares):
    """32 heads over 8: what a block joins one part after the other weighs against short prefixes."""
    assert longer_steps_share([n], [length], [tokens] * n, 4, 8) is shares


def test_nothing_to_share():
    for sizes, lengths, tokens in (([3], [0], [1, 5, 0]), ([1, 1], [64, 64], [700, 0]), ([1], [4096], [0])):
        assert longer_steps_share(sizes, lengths, tokens, 4, 8) is False
        assert single_tokens_share(sizes, [0] * len(sizes), 4096) is False


def test_lines_that_are_moved_out_of_the_way(monkeypatch):
    """As the tests of small cases do."""
    from kernel_rush_kawk_b200.cache import prefix

    monkeypatch.setattr(prefix, "JOIN_STEPS", -1e9)
    assert longer_steps_share([3], [0], [1, 5, 0], 4, 8) is True
    monkeypatch.setattr(prefix, "JOIN_STEPS", 1e9)
    assert longer_steps_share([64], [8192], [4] * 64, 4, 8) is False
