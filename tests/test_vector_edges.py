"""dedup.vector_edges where 4 and 8 bits say little about a vector: the pairs it keeps have to be those of the vectors themselves.
On the CPU (the operators from their definitions) and, marked gpu, on the engine."""
import os
import sys

import numpy as np
import pytest
import torch

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
from map_neo_amd import dedup as D  # noqa: E402
from test_vectors_path import VectorBackend  # noqa: E402


@pytest.fixture(params=["cpu", pytest.param("gpu", marks=pytest.mark.gpu)])
def backend(request):
    return VectorBackend() if request.param == "cpu" else request.getfixturevalue("engine")


def _true_cosines(x):
    x = x.double()
    n = x / x.norm(dim=1, keepdim=True)
    c = n @ n.T
    return c[np.tril_indices(len(x), -1)].numpy(), np.tril_indices(len(x), -1)


def _pairs(backend, x, t):
    u, v = D.vector_edges(backend, x.to(backend.device), t)
    return list(zip(u.cpu().tolist(), v.cpu().tolist()))


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("dim,big", [(1024, 130), (4096, 250), (4096, 260)])
def test_one_column_that_outweighs_the_others(backend, dim, big, dtype):
    """rows of +-1 but for a common column that sets the step of the 8-bit codes: the others become 0 or a whole step"""
    x = torch.randint(0, 2, (8, dim), generator=torch.Generator().manual_seed(0)).float() * 2 - 1
    x[:, 0] = big
    x = x.to(dtype)
    c, (u, v) = _true_cosines(x)
    assert c.max() < 0.97 and c.min() > 0.9
    assert _pairs(backend, x, 0.98) == []
    assert _pairs(backend, x, c.min() - 0.005) == list(zip(u, v))
    cut = np.sort(c)[13:15].mean()                               # between two pairs
    assert np.abs(c - cut).min() > 1e-9 and 0 < (c > cut).sum() < 28
    assert _pairs(backend, x, cut) == list(zip(u[c > cut], v[c > cut]))


@pytest.mark.parametrize("many", [False, True])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
def test_pairs_on_both_sides_of_the_threshold(backend, dtype, many):
    """cosines closer together than 8 bits can tell: 0.9 +- 10^-3 .. 10^-5, evenly sized columns; beside few other pairs, and
    beside a group of equal rows (more pairs than rows), one of them above and one below the threshold to all others"""
    g = torch.Generator().manual_seed(5)
    x = torch.randn(60, 512, generator=g, dtype=torch.float64)
    x /= x.norm(dim=1, keepdim=True)
    for k in range(30):
        c = 0.9 + (-1) ** k * 10.0 ** (-3 - 2 * k / 29)
        e = torch.randn(512, generator=g, dtype=torch.float64)
        e -= (e @ x[k]) * x[k]
        x[30 + k] = c * x[k] + np.sqrt(1 - c * c) * e / e.norm()
    if many:
        y = x[:1].repeat(20, 1)
        y[3], y[4] = x[30 + 4], x[30 + 5]
        x = torch.cat([y, x])
    x = (x * 3.7).to(dtype)
    c, (u, v) = _true_cosines(x)
    assert np.abs(c - 0.9).min() > 1e-9 and ((c >= 0.9).sum() > len(x)) == many
    assert _pairs(backend, x, 0.9) == list(zip(u[c >= 0.9], v[c >= 0.9]))
