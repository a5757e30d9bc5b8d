"""Distillation kernels on rows with extreme logits."""
import pytest
import torch

from distillation_extremes import check_lowest, check_masked_vocabulary, check_offset
from test_distillation_gpu import TYPES

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("rest", [False, True])
@pytest.mark.parametrize("tau,alpha", [(1.0, 1.0), (1.0, 0.5), (2.0, 0.5), (1.5, 1.0)])
def test_common_offset(tau, alpha, rest):
    check_offset(tau, rest, alpha, DEV)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rest", [False, True])
@pytest.mark.parametrize("alpha", [1.0, 0.5])
def test_rows_of_the_lowest_value(alpha, rest, dtype):
    check_lowest(rest, alpha, DEV, dtype)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rest", [False, True])
def test_vocabulary_masked_by_the_lowest_value(rest, dtype):
    check_masked_vocabulary(rest, DEV, dtype)
