"""The loops around the page operators over the reference, and what goes wrong without their rules."""
import pytest

from oracle import turn
from turn_loops import pages_back_beside_forked_rows, refused_fork_and_retry, rows_that_get_shorter

LISTS = lambda f: lambda *a: [x.tolist() if hasattr(x, "tolist") else x for x in f(*a)]
FORK, FREE = LISTS(turn.fork_rows), LISTS(turn.free_rows)


def test_a_refused_fork_is_not_taken():
    refused_fork_and_retry(FORK, FREE)


def test_a_loop_that_takes_the_count_of_a_refused_fork_loses_pages():
    with pytest.raises(AssertionError, match="a page is lost"):
        refused_fork_and_retry(FORK, FREE, took=lambda left: True)


def _by_hand(s, row):
    for page in s.table[row][:s.pages_of(s.lens[row])]:
        s.free[s.num] = page
        s.num += 1
    return True


def test_pages_that_other_rows_hold_stay_off_the_list():
    pages_back_beside_forked_rows(FORK, FREE)


def test_pages_returned_by_hand_beside_a_fork_are_held_and_free():
    with pytest.raises(AssertionError, match="held and free"):
        pages_back_beside_forked_rows(FORK, FREE, by_hand=_by_hand)


def test_rows_that_get_shorter_give_their_pages_back():
    rows_that_get_shorter(FORK, FREE)


def test_pages_behind_a_lowered_length_are_lost_by_themselves():
    with pytest.raises(AssertionError, match="a page is lost"):
        rows_that_get_shorter(FORK, FREE, give_back=False)
