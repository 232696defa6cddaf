"""GPU tests of log probabilities of long rows that begin anywhere between two 16-byte boundaries, with NaN in all elements that are no row's: rows that
fill whole units of 16 KB when they begin on a boundary, and reach into one more when they do not."""
import math

import pytest
import torch

from augur_v100_b200 import host
from test_gpu_token_logprobs import _check

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def stream():
    torch.cuda.set_device(0)
    s = host.Stream(0)
    yield s
    s.close()


@pytest.mark.parametrize("kind", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("k", [0, 20, 32])
@pytest.mark.parametrize("rows,n,stride,offset", [(3, 4096, 4097, 0), (5, 8192, 8193, 3), (450, 8192, 8195, 1), (8, 8191, 8192, 1), (9, 16384, 16391, 7), (700, 1025, 1031, 5),
                                                  (2, 100003, 100003, 2), (61, 65536, 65537, 0), (450, 24575, 24577, 0)])
def test_rows_that_begin_anywhere(stream, rows, n, stride, offset, k, kind):
    g = torch.Generator(device="cuda:0").manual_seed(rows + n + offset)
    memory = torch.full((rows * stride + offset + 16,), math.nan, dtype=kind, device="cuda:0")
    x = memory.as_strided((rows, n), (stride, 1), offset)
    x.copy_(torch.randn((rows, n), generator=g, device="cuda:0") * 3)
    _check(stream, x, torch.randint(n, (rows,), generator=g, device="cuda:0", dtype=torch.int32), k)


@pytest.mark.parametrize("kind", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n,stride", [(8192, 8193), (100003, 100005)])
def test_hard_orders_that_begin_anywhere(stream, n, stride, kind):
    index = torch.arange(n, device="cuda:0")
    ramp = torch.linspace(-4, 4, n, device="cuda:0")
    rows = [ramp, ramp.flip(0), torch.zeros(n, device="cuda:0"), (index % 7).float(), torch.where(index >= n - 3, 9.0, 0.0), torch.where(index < 3, 9.0, 0.0),
            torch.where(index == n - 1, 0.0, -math.inf), torch.where(index == 0, 0.0, -math.inf)] * 4
    memory = torch.full((len(rows) * stride + 16,), math.nan, dtype=kind, device="cuda:0")
    x = memory.as_strided((len(rows), n), (stride, 1), 1)
    x.copy_(torch.stack(rows))
    _check(stream, x, torch.full((len(rows),), n - 1, dtype=torch.int32, device="cuda:0"), 32)
