"""The small decoder's host side: drafts and page tables."""

import pytest
import torch

from sonic_sampler_b200.decode import drafts_from_history, main, page_table


def test_drafts_follow_the_last_occurrence_of_the_newest_token():
    assert drafts_from_history([[1, 2, 3, 1, 4, 5, 1]], 2) == [[4, 5]]
    assert drafts_from_history([[7, 8, 7]], 3) == [[8, 7, 7]]
    assert drafts_from_history([[1, 2, 3], [5]], 2) == [[3, 3], [5, 5]]


def test_page_tables_hand_every_page_out_once():
    table = page_table(3, 33, 16, 10, "cpu")
    assert table.shape == (3, 3) and table.dtype == torch.int32
    assert len(set(table.view(-1).tolist())) == 9 and int(table.max()) < 10
    with pytest.raises(ValueError, match="need 9 pages"):
        page_table(3, 33, 16, 8, "cpu")


def test_the_command_refuses_empty_work():
    with pytest.raises(SystemExit):
        main(["--requests", "0"])
    with pytest.raises(SystemExit):
        main(["--lookahead", "-1"])
