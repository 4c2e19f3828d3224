"""as_sample_tokens' argument checks (answered on the host) and the oracle's sampler."""

import math

import numpy as np
import pytest
import torch

from agentserve_b200 import _native as N
from agentserve_b200 import ops
from oracle import sampling as OS


@pytest.fixture(scope="module")
def lib():
    if not N.LIB_PATH.exists():
        from agentserve_b200.build import build
        build()
    return N.load()


def test_bad_arguments_are_refused_before_any_launch(lib):
    def call(out=None, logits=None, stride=100, u=None, t=None, rows=4, vocab=100,
             dtype=N.AS_DTYPE_BF16):
        return lib.as_sample_tokens(out, None, logits, stride, u, t, None, None, None, rows,
                                    vocab, dtype, None)
    assert call(dtype=9) == N.AS_ERR_INVALID_ARG and "dtype" in N.last_error()
    assert call(stride=99) == N.AS_ERR_INVALID_ARG
    assert call(rows=-1) == N.AS_ERR_INVALID_ARG
    assert call(vocab=0) == N.AS_ERR_INVALID_ARG
    assert call() == N.AS_ERR_INVALID_ARG and "null pointer" in N.last_error()
    assert call(vocab=(1 << 20) + 1, stride=1 << 21) == N.AS_ERR_UNSUPPORTED
    assert call(out=64, logits=65, u=64, t=64) == N.AS_ERR_INVALID_ARG
    assert "aligned" in N.last_error()
    assert call(rows=0) == N.AS_OK


def test_cpu_tensors_are_refused():
    with pytest.raises(RuntimeError):
        ops.sample_tokens(torch.zeros(2, 8), torch.zeros(2), torch.ones(2))


def test_oracle_keeps_prefixes_of_one_order():
    row = np.array([1.0, 3.0, 3.0, 2.0, -np.inf, np.nan], dtype=np.float32)
    kept, w = OS.kept_tokens(row, 1.0, top_k=2)
    assert kept == [1, 2] and w == [1.0, 1.0]
    assert OS.kept_tokens(row, 1.0, top_k=1)[0] == [1]
    assert OS.kept_tokens(row, 0.0)[0] == [1]
    # 1, 1, e^-1, e^-2, e^-3 (NaN counts as 0), nothing for -inf: 2.553 in all, so a
    # share of 0.4 (1.02) takes both maxima and 0.39 (0.996) one
    assert OS.kept_tokens(row, 1.0, top_p=0.39)[0] == [1]
    assert OS.kept_tokens(row, 1.0, top_p=0.4)[0] == [1, 2]
    assert OS.kept_tokens(row, 1.0, top_p=0.41)[0] == [1, 2]
    assert OS.kept_tokens(row, 1.0, min_p=0.2)[0] == [1, 2, 3]
    t, lp = OS.sample(row, 0.5, 1.0, top_k=2)
    assert t == 2 and math.isclose(lp, math.log(0.5))
