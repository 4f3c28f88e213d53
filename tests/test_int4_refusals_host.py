"""Calls of the 4-bit row cache that are refused before anything runs (no GPU)."""
import pytest
import torch

from logitfill_amd import _native
from logitfill_amd.packed import int4
from logitfill_amd.packed.reference import reference_attention
from logitfill_amd.qwen2 import attach_packed
from tests.test_int4_host import _args, _layer


@pytest.mark.parametrize("scaling", [float("nan"), float("inf"), -float("inf")])
def test_a_scaling_that_is_not_finite(scaling):
    """NaN became the smallest factor: finite outputs, every row's weight equal."""
    assert _native.load().lf_int4_attention(_layer(), _args(scaling=scaling), None) == _native.LF_E_SHAPE

    class Manager:
        batch_size, n_q, n_kv, head_dim, device, top_pages = 1, 2, 1, 64, torch.device("cpu"), 0
        layers = [None]
    for s in (scaling, torch.tensor(scaling)):
        with pytest.raises(ValueError, match="finite"):
            int4.int4_attention(Manager, 0, torch.empty(1, 2, 1, 64), None, None, s)


def test_the_dense_path_of_packed_pages():
    """It failed at the first decode step, the prompt committed."""
    manager = int4.Int4KVManager.__new__(int4.Int4KVManager)
    with pytest.raises(ValueError, match="int4_attention"):
        attach_packed(None, manager, reference_attention)


def test_many_row_rule_by_the_work_in_front_of_every_row():
    """Rows add partial sums and their merge: short histories stay with the general kernel, however many rows there are (four
    sequences of 2K tokens, 1 024 queries, groups of 128: 277 us by the many-row kernel, 186 without)."""
    for args, want in (((7, 1024, 4, 128, 128, torch.bfloat16, [2048] * 4), False), ((7, 512, 4, 128, 128, torch.bfloat16, [4096] * 4), False),
                       ((7, 512, 4, 128, 128, torch.bfloat16, [16384] * 4), True), ((4, 512, 8, 128, 32, torch.bfloat16, [4096] * 4), True),
                       ((7, 256, 2, 64, 64, torch.bfloat16, [32768]), True), ((7, 1024, 2, 64, 64, torch.bfloat16, [2048] * 4), False)):
        assert int4._many_rows(*args) is want, args
