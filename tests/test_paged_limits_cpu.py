"""What the entry points over a paged cache refuse at their limits, before anything is launched.  No GPU needed."""

import pytest

from flash_colsum_b200 import _cabi
from test_paged_cpu import attend


@pytest.mark.parametrize("k", [2 ** 26 + 1, 2 ** 27, 2 ** 31 - 1])
def test_lists_that_the_attention_cannot_count_are_refused(k):
    assert attend(k=k) < 0
    assert "at most 67108864 pages" in _cabi.last_error()
