"""The loops around the page operators over the reference, and what goes wrong without their rules."""
import pytest

from oracle import turn
from turn_loops import refused_fork_and_retry

LISTS = lambda f: lambda *a: [x.tolist() if hasattr(x, "tolist") else x for x in f(*a)]
FORK, FREE = LISTS(turn.fork_rows), LISTS(turn.free_rows)


def test_a_refused_fork_is_not_taken():
    refused_fork_and_retry(FORK, FREE)


def test_a_loop_that_takes_the_count_of_a_refused_fork_loses_pages():
    with pytest.raises(AssertionError, match="a page is lost"):
        refused_fork_and_retry(FORK, FREE, took=lambda left: True)
