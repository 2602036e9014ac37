"""CPU: the dealing out of work over tiles of 8 and 32 rows, which the attention of few rows takes beside those of 16 (test_paged_rules_cpu)."""
import pytest

from test_paged_rules_cpu import rules  # noqa: F401  (a fixture)
from test_paged_rules_cpu import test_a_tile_holds_whole_tokens_and_every_head_once as whole_tokens_and_every_head_once
from test_paged_rules_cpu import test_every_unit_has_its_place as every_unit_has_its_place


@pytest.mark.parametrize("rows", [8, 32])
@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (12, 12), (32, 8), (7, 1), (40, 2), (20, 1), (64, 2), (33, 1), (300, 1)])
def test_small_tiles_hold_whole_tokens_and_every_head_once(rules, heads, kv_heads, rows):  # noqa: F811
    whole_tokens_and_every_head_once(rules, heads, kv_heads, rows, 1)


@pytest.mark.parametrize("causal", [0, 1])
@pytest.mark.parametrize("heads,kv_heads,rows", [(12, 12, 8), (32, 8, 8), (40, 1, 8), (5, 1, 8), (12, 12, 32), (32, 8, 32), (7, 1, 32), (34, 2, 32), (150, 1, 32)])
def test_every_unit_of_small_tiles_has_its_place(rules, heads, kv_heads, rows, causal):  # noqa: F811
    every_unit_has_its_place(rules, heads, kv_heads, rows, 1, 128, causal, 0)
