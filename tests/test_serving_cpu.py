"""CPU: the engine's own proposer of drafts."""
import pytest


@pytest.mark.parametrize("tokens,most,want", [
    ([1, 2, 3, 1, 2], 3, [3, 1, 2]), ([1, 2, 3, 1, 2], 1, [3]), ([7, 7, 7, 7], 2, [7]), ([1, 2, 3], 4, []), ([5], 4, []), ([], 4, []),
    ([1, 2, 9, 3, 2, 8, 1, 2], 2, [9, 3]), ([1, 2, 3, 1, 2], 0, []),
])
def test_lookup_drafts(tokens, most, want):
    from omlx_exl3_b200.serving import lookup_drafts
    assert lookup_drafts(tokens, most) == want
