"""Settings that a sampled step could not stage: refused when they are made, and so at submit,
or not read at all (greedy requests)."""

import numpy as np
import pytest

from agentserve_b200 import B200Engine, Request, SamplingParams
from agentserve_b200 import sampling as S
from tests.test_engine_host import FAKE_CFG, E


@pytest.mark.parametrize("top_k", [None, "many", float("inf"), float("nan"), [3]])
def test_a_top_k_that_is_no_number_is_refused(top_k):
    with pytest.raises(ValueError, match="top_k"):
        SamplingParams(0.7, top_k=top_k)

    class Sampled(E.HistoryModelForB200):
        def prefill_paged_sampled(self, *args):
            raise AssertionError("no step runs here")

    engine = B200Engine(FAKE_CFG, model=Sampled(), num_cache_blocks=64, per_request_sampling=True)
    bad = Request(prompt="b", token_ids=[1, 2], max_tokens=2, temperature=0.7, top_k=top_k)
    with pytest.raises(ValueError, match="top_k"):
        engine.submit(bad)
    assert not engine._incoming


def test_whole_numbers_of_any_type_and_size_are_staged():
    out = np.zeros((S.STAGED, 4), dtype=np.int32)
    S.stage(out, [SamplingParams(1.0, k) for k in (np.int64(7), 10 ** 30, -10 ** 30, 5.0)], [0.5] * 4)
    assert out[1].tolist() == [7, 2 ** 31 - 1, 0, 5]


def test_a_greedy_request_stages_none_of_its_other_settings():
    """A batch holds greedy and sampled requests; what a greedy one carries is not used."""
    odd = [SamplingParams(0.0, None, None, None), SamplingParams(-1.0, 3, 0.5, 0.5),
           SamplingParams(float("nan"), "x", float("nan"), 7.0)]
    out = np.full((S.STAGED, 5), 9, dtype=np.int32)
    S.stage(out, odd + [SamplingParams(0.5, 7, 0.25, 0.125)], [0.5, 0.25, 0.125, 0.75])
    f = out.view(np.float32)
    assert f[0].tolist() == [0.0, 0.0, 0.0, 0.5, 0.0]
    assert out[1].tolist() == [0, 0, 0, 7, 0]
    assert f[2].tolist() == [1.0, 1.0, 1.0, 0.25, 1.0]
    assert f[3].tolist() == [0.0, 0.0, 0.0, 0.125, 0.0]
    assert f[4].tolist() == [0.5, 0.25, 0.125, 0.75, 0.0]
