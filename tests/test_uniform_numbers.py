"""Numbers of [0, 1) that float32 would round up to one, given to the verification of drafts."""
import numpy as np
import pytest
import torch

from dlgo_amd.sampling import SamplerConfig
from dlgo_amd.sampling.sampler import _below_one

TOP = 1 - 2.0 ** -24


def test_they_stay_below_one():
    got = _below_one([[0.0, 0.25, 1 - 2.0 ** -30], [], [1 - 2.0 ** -53, TOP, 1 - 2.0 ** -23]], 6)
    assert got.dtype == np.float32 and got.tolist() == [0.0, 0.25, TOP, TOP, TOP, 1 - 2.0 ** -23]


@pytest.mark.gpu
def test_a_sure_draft_is_kept_and_the_last_token_of_weight_is_drawn():
    """One token has all the weight: kept for every number below one.  Beside it, a draw at the very end of [0, 1)."""
    from dlgo_amd.sampling.sampler import Sampler
    s = Sampler(5000, "cuda:0")
    logits = torch.full((3, 5000), -1000.0, device="cuda:0")
    logits[0, 7] = logits[1, 9] = 0.0
    logits[2, 11:4000] = 0.0
    alone = SamplerConfig(temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, repetition_penalty=1.0)
    for u in (TOP, 1 - 2.0 ** -30, 1 - 2.0 ** -53):
        assert s.verify(logits, [[7], []], [alone] * 2, [[u, u], [u]]) == ([1, 0], [9, 3999])
