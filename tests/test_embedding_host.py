"""Argument checks of the embedding entry points, on the CPU."""

import pytest
import torch

from causal_tuner_b200 import _lib
from causal_tuner_b200.kernels.embedding_cuda import embed_tokens, embedding_gradient


def test_entry_points_check_their_arguments():
    library = _lib.load()
    forward, gradient = library.ct_embedding_forward, library.ct_embedding_gradient
    assert forward(None, None, None, 0, 10, 8, 1.0, 0, 0, None) == _lib.OK
    assert forward(None, None, None, 4, 10, 8, 1.0, 0, 0, None) == _lib.ERR_ARG
    assert forward(None, None, None, -1, 10, 8, 1.0, 0, 0, None) == _lib.ERR_ARG
    assert forward(None, None, None, 4, 10, 8, 1.0, 0, 5, None) == _lib.ERR_ARG
    assert gradient(None, 8, None, None, 4, 0, 8, 1.0, -1, 0, 0, None, None) == _lib.OK
    assert gradient(None, 8, None, None, 4, 10, 8, 1.0, -1, 0, 0, None, None) == _lib.ERR_ARG
    assert gradient(None, 7, None, None, 4, 10, 8, 1.0, -1, 0, 0, None, None) == _lib.ERR_ARG
    some = torch.zeros(1).data_ptr()
    assert gradient(some, 8, some, some, 1 << 31, 10, 8, 1.0, -1, 0, 0, some, None) == _lib.ERR_UNSUPPORTED


def test_workspace():
    size = _lib.load().ct_embedding_gradient_workspace
    # two lists of 1000 tokens, 11 run starts, 32 pieces x 2 rows of 16 floats
    assert size(1000, 10, 16) == 2 * 4096 + 256 + 4096
    # above 1024 tokens four lists and the blocks' histograms
    assert size(20000, 10, 16) == 4 * 80128 + 8 * 256 * 4 + 256 + 625 * 2 * 64 + 128


def test_no_cpu_path():
    ids, weight = torch.zeros(3, dtype=torch.int64), torch.zeros(4, 8)
    with pytest.raises(RuntimeError, match="no CPU path"):
        embed_tokens(ids, weight)
    with pytest.raises(RuntimeError, match="no CPU path"):
        embedding_gradient(torch.zeros(3, 8), ids, 4)
