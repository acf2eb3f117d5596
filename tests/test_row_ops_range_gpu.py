"""The language-model row operators at the ends of their ranges: subnormal, tiny and huge numbers,
neighbouring numbers, NaN in biases, workspaces on the least alignment that is asked for.

Against the 64-bit forms, with the tolerances of test_row_ops_gpu.py.
"""
import pytest
import torch

from tests import row_ops_ref as ref
from tests.test_row_ops_gpu import FOLD, T, check_route, check_sample, near, rand  # noqa: F401  (T: the fixture)

pytestmark = pytest.mark.gpu


# --------------------------------------------------------------- sampling


def subnormals(least, most):
    """f32 numbers of the bits `least` to `most`."""
    return torch.arange(least, most + 1, dtype=torch.int32, device="cuda").view(torch.float32)


def test_sample_threshold_among_subnormals_beside_zeros(T):
    """A range of the search that ends just below the zeros: the key between them and the largest
    negative number is no number's, and none may be counted under it."""
    g = torch.Generator(device="cuda").manual_seed(2)
    rows = []
    for zeros, below in ((5000, 3000), (1100, 1100), (9000, 8000)):
        row = torch.full((20000,), -9.0, device="cuda")
        row[:zeros] = 0.0
        row[:zeros:3] = -0.0
        row[zeros] = subnormals(0x3ff, 0x3ff)
        row[zeros + 1:zeros + 1 + below] = -subnormals(1, 1000).repeat(9)[:below]
        rows.append(row[torch.randperm(20000, device="cuda", generator=g)])
    logits = torch.stack(rows)
    u = torch.tensor([0.1, 0.6, 0.97], device="cuda")
    for k in (1, 2, 1100, 1101, 1102, 1500, 2200, 5001, 5002, 5500, 9001, 9002, 12000):
        check_sample(T, logits, u, top_k=k)
        check_sample(T, logits, u, top_k=k, top_p=0.7)
    # Weights of 1 but for the -9: masses in the same ranges.
    for p in (0.2, 0.5, 0.63, 0.64, 0.9, 0.99):
        check_sample(T, logits, u, top_p=p)
