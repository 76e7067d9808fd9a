"""thin_cache_attention where values and scales of some rows' tokens are not others':
against the 64-bit definition, within oracle.attend.allowed() of what each row sees."""
import math

import pytest
import torch

from tests.helpers import gen
from tests.test_gpu_cache import HALVES, Cache, queries

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("d", [96, 128, 208, 256])
def test_nan_values_among_the_first_keys(gpu, dtype, d):
    """Many rows that begin with the sequence: NaN values of the first 32 keys, in
    dims of every wavefront's, reach the rows from their key on and no earlier one."""
    c = Cache(gpu, 3, 3, 16, 2, d, d)
    keys = (0, 5, 16, 31)
    for i in range(3):
        for n, j in enumerate(keys):
            c.host[1][c.table[i, j // 16].long(), n % 2, j % 16, (n + i) * (d // 8) + d // 4::d // 2] = 0x7F
    c.dev = [x.to(gpu) for x in c.host]
    q = queries(3, 40, 4, d, HALVES[dtype], 1)
    got = c.attend(q, torch.tensor([40, 41, 48], dtype=torch.int32))
    nan = torch.isnan(got.cpu())
    assert nan[0, 0, :2].any() and not nan[0, :5, 2:].any() and nan[0, 5:, 2:].any(2).all()
    c.attend(q, torch.tensor([40, 40, 40], dtype=torch.int32), torch.tensor([40, 33, 39], dtype=torch.int32))
