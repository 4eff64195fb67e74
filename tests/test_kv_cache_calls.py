"""KV caches by handle, without a GPU: which host-side calls are taken, which are refused, and that a refused call leaves nothing behind."""
import types

import pytest
import torch

from seed_amd.kv_cache import KVCache


# ------------------------------------------------------------------------------------------------ rows of a call
@pytest.mark.parametrize("rows,tokens", [(8, 3), (10, 4), (12, 5), (7, 8), (4, 0), (4, -2)])
def test_rows_that_tokens_do_not_divide_are_refused(rows, tokens):
    """tokens=3 asks for slots of three rows: eight rows are not two slots of four."""
    with pytest.raises(ValueError, match="do not divide"):
        KVCache._batch(types.SimpleNamespace(slots=8), "append", rows, 0, tokens)


@pytest.mark.parametrize("rows,tokens,lens,want", [(8, 4, 0, (2, 4)), (8, 1, 0, (8, 1)), (3, 3, 0, (1, 3)), (8, None, 0, (4, 2)),
                                                   (6, None, torch.zeros(3, dtype=torch.int32), (3, 2)), (6, 2, torch.zeros(4, dtype=torch.int32), (3, 2))])
def test_slots_and_tokens_of_a_call(rows, tokens, lens, want):
    assert KVCache._batch(types.SimpleNamespace(slots=8 if tokens else 4), "append", rows, lens, tokens) == want
