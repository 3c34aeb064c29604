"""Row tiles with rows that belong to no query hold what an earlier kernel left in shared memory: it changes nothing."""
import pytest
import torch

import operator_definitions as defs

pytestmark = pytest.mark.gpu

k = pytest.importorskip("krea2_hrx_b200")
from krea2_hrx_b200 import ops  # noqa: E402


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("q_len,kv_len,heads", [(400, 700, 3), (400, 700, 5), (90, 4000, 7), (400, 300, 24), (1, 700, 48)])
def test_rows_of_nobody(dim, q_len, kv_len, heads):
    g = torch.Generator(device="cuda").manual_seed(heads)
    q, key, value = (torch.randn(shape, generator=g, device="cuda").to(torch.bfloat16) for shape in
                     ((1, q_len, heads, dim), (1, kv_len, 1, dim), (1, kv_len, 1, dim)))
    # full tiles of NaN (and of infinities) on every SM, whose rows and outputs stay behind
    many = 256 * torch.cuda.get_device_properties(0).multi_processor_count
    outs = []
    for left in (0.0, float("nan"), float("inf")):
        before = torch.full((1, many, 1, dim), left, dtype=torch.bfloat16, device="cuda")
        ops.cross_attention(before, key, value, torch.empty_like(before))
        outs.append(torch.full_like(q, 9.0))
        ops.cross_attention(q, key, value, outs[-1])
    defs.check_cross(outs[0], q, key, value, dim ** -0.5)
    assert torch.equal(outs[0], outs[1]) and torch.equal(outs[0], outs[2])
    assert k.device_status() == 0
