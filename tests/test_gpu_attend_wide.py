"""The tests of tests/test_gpu_attend.py with page tables that have room for more than 1024 keys.  A short table has the
one-launch form of few rows do the work whatever the call brings; with a wide one chunks go through the form of chunks,
and single tokens through the one that cuts and joins."""
import numpy as np
import pytest

import tests.test_gpu_attend as short
from tests.test_gpu_attend import (  # noqa: F401
    be, test_bad_tables_raise_a_fault_and_touch_nothing_else, test_chunks, test_heads_that_are_no_power_of_two, test_many_sequences,
    test_recorded_and_replayed_with_growing_lengths, test_released_pages_behind_the_window_are_not_looked_up, test_results_repeat_bit_for_bit,
    test_row_offsets_that_name_rows_twice, test_rows_without_keys_and_rows_of_nobody, test_scales, test_scores_far_apart_and_queries_of_all_sizes,
    test_single_tokens, test_the_output_may_be_the_query, test_what_is_masked_does_not_reach_a_row, test_work_queued_on_another_stream_is_waited_for)

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def wide_tables(monkeypatch):
    made = short.make_case

    def make(*args, **kw):
        c = made(*args, **kw)
        c["table"] = np.pad(c["table"], ((0, 0), (0, 1100 // c["page"] + 1)), constant_values=-1)
        return c

    monkeypatch.setattr(short, "make_case", make)
