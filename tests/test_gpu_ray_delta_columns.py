"""The delta rule for every width of keys and values: wavefronts that hold some columns, all, or none."""
import pytest
import torch

from ray_oracle import ray_set
from test_gpu_ray_delta import check

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("dv", list(range(8, 129, 8)))
def test_value_columns(dv, dtype):
    check(ray_set([35, 16]), 1, 2, 16, dv, dtype, seed=dv, start=True)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("dk", list(range(8, 129, 8)))
def test_key_columns(dk, dtype):
    check(ray_set([35, 16]), 1, 1, dk, 80, dtype, seed=dk, start=True)
