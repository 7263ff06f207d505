"""Gradients of B and C where few channels share them: a sum of few terms shows the rounding of each.  As ``test_selective_scan``, at its
tolerances, in which a bfloat16 result has one rounding to its type and what float32 arithmetic adds."""

import pytest
import torch

from tests import test_gpu_selective as S

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("T,R,W,N,G,layout,masks", [
    (1, 1, 9, 8, 9, "columns", "ragged"),
    (3, 39, 1, 16, 1, "dense", "done"),
    (2, 185, 19, 8, 19, "batch", "ragged"),
    (1, 415, 13, 16, 1, "batch", "done"),
    (24, 25, 7, 10, 7, "dense", ""),
    (2, 132, 3, 32, 3, "dense", "ragged"),
    (2, 60, 66, 4, 33, "columns", "done ragged"),
    (40, 12, 6, 2, 2, "dense", "done"),
])
@pytest.mark.parametrize("full", [True, False])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_sums_of_few_terms(T, R, W, N, G, layout, masks, full, dtype):
    S.test_selective_scan(T, R, W, N, G, dtype, layout, masks, full)
