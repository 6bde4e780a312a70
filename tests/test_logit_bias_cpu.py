"""What a request's biases may be: one value a token, tokens whole numbers."""

import numpy as np
import pytest
import torch

from aspire_amd.logits_processor import LogitBias


def test_tokens_of_any_integer_type():
    b = LogitBias([{np.int64(7): 1, 2: np.float32(0.5), True: 2.0, 9.0: 3.0}, {torch.tensor(4): torch.tensor(1.5)}], "cpu")
    assert b.ids.tolist() == [1, 2, 7, 9, 4] and b.values.tolist() == [2.0, 0.5, 1.0, 3.0, 1.5] and b.indptr.tolist() == [0, 4, 5]


@pytest.mark.parametrize("bad", [{1.5: 1.0}, {1: 1.0, 1.5: 2.0}, {torch.tensor(3): 1.0, 3: 2.0}, {torch.tensor(3): 1.0, torch.tensor(3): 2.0}, {"3": 1.0},
                                 {float("nan"): 1.0}, {float("inf"): 1.0}, {None: 1.0}, {3: None}])
def test_what_is_no_token_or_twice_one_is_refused(bad):
    """Of two values of one token either would count, by chance."""
    with pytest.raises((ValueError, TypeError, OverflowError)):
        LogitBias([{}, bad], "cpu")
