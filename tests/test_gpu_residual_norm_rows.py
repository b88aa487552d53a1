"""Short float32 rows, so many that the forward pass takes more channels a thread than the backward pass: a slice of them in float64."""
import pytest
import torch

from tests.test_gpu_residual_norm import exact, hold, make, run

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize('rows,c', [(2500003, 8), (1600001, 13), (320007, 64), (200003, 100), (160001, 128), (87001, 230), (79003, 256), (78001, 256)])
def test_short_rows(rows, c):
    gen = torch.Generator().manual_seed(c)
    d = make(gen, (rows, c), torch.float32, torch.float32)
    got = run(d, 'silu', wrt=('input', 'residual', 'gate'))
    for part in (slice(0, 70), slice(rows // 2, rows // 2 + 70), slice(rows - 70, rows)):
        few = {k: v[part] if v is not None and v.dim() > 1 else v for k, v in d.items()}
        want = exact(few, 'silu')
        hold({k: v[part] for k, v in got.items()}, want, 70)
