"""What the rotary operators keep of a call's sections and frequencies: numbers, by their values."""
import gc
import weakref

import pytest
import torch

from inductor_x_b200 import ops


def call(sections, frequencies):
    """Refused as host memory is, behind the plan."""
    with pytest.raises(ValueError, match="CUDA|cuda|device"):
        ops.axial_rotary(torch.empty(1, 1, 3, 16), None, torch.zeros(len(sections), 3, dtype=torch.int64), sections, frequencies=frequencies)


def test_frequencies_in_a_tensor_are_kept_by_value():
    f = torch.tensor([0.5, 0.25, 0.125, 3.0], dtype=torch.float64)
    before = ops._rotary_plan.cache_info()
    for _ in range(3):
        call([3, 1], f)
        call(torch.tensor([3, 1]), list(f))
        call((3, 1), tuple(f.tolist()))
    after = ops._rotary_plan.cache_info()
    assert after.misses == before.misses + 1 and after.hits == before.hits + 8
    f[0] = 0.75
    call([3, 1], f)
    assert ops._rotary_plan.cache_info().misses == after.misses + 1
    plan = ops._rotary_plan((3, 1), 10000.0, "shared", (0.75, 0.25, 0.125, 3.0))
    assert list(plan[3]) == f.tolist() and list(plan[2]) == [3, 1]
    held = weakref.ref(f.untyped_storage())
    del f
    gc.collect()
    assert held() is None


def test_sections_are_whole_numbers_whatever_was_asked_before():
    call([5, 2], None)
    with pytest.raises(TypeError):
        call([5.0, 2.0], None)
