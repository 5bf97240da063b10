"""Arguments of the attention-side calls that are refused before any GPU is needed."""

import ctypes as C

import pytest
import torch

from klearu_b200 import _lib
from klearu_b200.attention import RopeTable, SeqBatch


@pytest.mark.parametrize("kw", [{"rot_dim": 0}, {"rot_dim": 3}, {"base": 0.0}, {"factor": -1.0}, {"scaling": "other"},
                                {"attention_factor": float("nan")}, {"scaling": "by_parts"},
                                {"scaling": "by_parts", "original_positions": 64, "low_turns": 4.0, "high_turns": 4.0}])
def test_rope_arguments(kw):
    with pytest.raises(ValueError):
        RopeTable(**{"rot_dim": 64, "max_positions": 16, **kw})


def test_batch_wants_gpu_tensors():
    with pytest.raises(ValueError):
        SeqBatch(torch.zeros(2, dtype=torch.int32), torch.zeros(1, dtype=torch.int32),
                 torch.zeros(1, 1, dtype=torch.int32), max_q=1)


def test_null_handles():
    lib = _lib.load()
    n = C.c_size_t()
    assert lib.kl_rope_create(None, 64, 16, None, 1.0, 0, None) == _lib.KL_EINVAL
    assert lib.kl_rope_destroy(None) == _lib.KL_EINVAL
    assert lib.kl_kv4_create(None, 1, 16, 1, 64, None) == _lib.KL_EINVAL
    assert lib.kl_kv4_destroy(None) == _lib.KL_EINVAL
    assert lib.kl_kv4_append(None, None, None, None, 0, None, None, None, None) == _lib.KL_EINVAL
    assert lib.kl_kv4_read(None, None, None, None) == _lib.KL_EINVAL
    assert lib.kl_kv4_attend_workspace(None, None, 1, 0, C.byref(n)) == _lib.KL_EINVAL
    assert lib.kl_kv4_attend(None, None, 1, None, None, 1.0, 0, None, 0) == _lib.KL_EINVAL
    assert lib.kl_norm_q8(None, None, 0, 1, None, 0, None, 1, 1, 0.0, 0, 0, None, 0, None, 0, None) == _lib.KL_EINVAL
    assert lib.kl_q8_linear_create(None, 1, 1, None, 1, None, None, None) == _lib.KL_EINVAL
    assert lib.kl_q8_linear_destroy(None) == _lib.KL_EINVAL
    assert lib.kl_q8_linear_forward(None, None, 16, None, 1, None, 0, 1, 0) == _lib.KL_EINVAL


def test_sizes_of_the_call_structs():
    """The ctypes mirrors have the C layout: four 8-byte fields and five of 4 bytes; three of 8."""
    assert C.sizeof(_lib.SeqBatchC) == 56 and C.sizeof(_lib.HeadRowsC) == 24
