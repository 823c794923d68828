"""The id of padding: below 0 none, up to what an int32 id of a table can be."""
import pytest
import torch


def test_padding_id(mc):
    """int64 ids past int32 arrive as 2**31 - 1, which as the id of padding would give them zeros in place of NaN."""
    table, ids = torch.zeros(10, 8), torch.zeros(2, 3, dtype=torch.int64)
    calls = (lambda p: mc.embedding_forward(table, ids, padding_id=p),
             lambda p: mc.embedding_backward(torch.zeros(2, 3, 8), ids, 10, padding_id=p))
    for call in calls:
        for bad in (2**31 - 1, 2**31, 2**40, 2**64 + 5):
            with pytest.raises(mc.McError) as e:
                call(bad)
            assert e.value.code == 5 and "padding_id must be below" in str(e.value)
        for good in (None, -1, -100, 0, 9, 10, 2**31 - 2):
            with pytest.raises(Exception) as e:  # the call goes on to what refuses the CPU
                call(good)
            assert "padding_id" not in str(e.value)
