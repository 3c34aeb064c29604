"""The norm's codes over the whole range of bf16: rows whose squares leave that of f32, on either side."""
import pytest
import torch

import operator_definitions as defs

pytestmark = pytest.mark.gpu

k = pytest.importorskip("krea2_hrx_b200")
from krea2_hrx_b200 import ops  # noqa: E402

NORM_ROUNDINGS = 60  # as in the tests of ordinary rows: squares, their additions, the root and the factor; powers of two are exact


def norm_codes(x, residual=None, eps=1e-5, total=None):
    rows, width = x.shape
    q = torch.empty((rows, -(-width // 16) * 16), dtype=torch.float8_e4m3fn, device="cuda")[:, :width]
    scales = torch.empty((rows, defs.groups(width)), device="cuda")
    ops.prepare_norm_fp8(x, None, q, scales, residual=residual, sum_out=total, eps=eps, weight_offset=1.0)
    return q, scales


# one warp, rows of single elements, one, two, three and eight runs of eight channels a thread
@pytest.mark.parametrize("rows,width", [(9, 96), (9, 129), (9, 1000), (9, 12345), (200, 2056), (200, 6144), (9, 16384), (9, 32768)])
@pytest.mark.parametrize("exponent,eps", [(-126, 0.0), (-90, 0.0), (-70, 0.0), (-55, 0.0), (-100, 2.0 ** -110), (-120, 2.0 ** -126), (50, 0.0), (60, 1e-5),
                                          (70, 1.0), (120, 1e-5), (124, 1e-5)])
def test_rows_whose_squares_leave_the_range_of_f32(rows, width, exponent, eps):
    """Ordinary rows between the tiny (or huge) ones keep their codes: a block takes each row by itself."""
    x = torch.randn((rows, width), generator=torch.Generator().manual_seed(width), dtype=torch.float64).clamp(-7, 7)
    x[::3] *= 2.0 ** exponent
    x[1::9] *= 2.0 ** (exponent // 2)
    x = x.cuda().to(torch.bfloat16)
    q, scales = norm_codes(x, eps=eps)
    want, _ = defs.norm_rows(x, None, None, eps, 1.0)
    defs.check_codes(q, scales, want, NORM_ROUNDINGS)


@pytest.mark.parametrize("width", [129, 6144])
@pytest.mark.parametrize("exponent", [-110, 120])
def test_a_residual_s_sum_outside_the_range_of_its_squares(width, exponent):
    g = torch.Generator().manual_seed(5)
    x, residual = ((torch.randn((160, width), generator=g, dtype=torch.float64) * 2.0 ** exponent).cuda().to(torch.bfloat16) for _ in range(2))
    want, want_sum = defs.norm_rows(x, residual, None, 0.0, 1.0)
    total = torch.empty_like(x)
    q, scales = norm_codes(x, residual, 0.0, total)
    assert torch.equal(total.cpu(), want_sum)
    defs.check_codes(q, scales, want, NORM_ROUNDINGS)


def test_one_large_value_in_a_row_of_ordinary_ones():
    x = torch.randn((4, 6144), generator=torch.Generator().manual_seed(6)).cuda().to(torch.bfloat16)
    x[0, 4000], x[1, 0], x[2, 77] = 3.0e38, -2.0 ** 65, 2.0 ** 127
    q, scales = norm_codes(x)
    want, _ = defs.norm_rows(x, None, None, 1e-5, 1.0)
    defs.check_codes(q, scales, want, NORM_ROUNDINGS)


def test_special_values_among_huge_and_tiny_ones():
    """A NaN reaches its row, an infinity leaves zeros beside itself, and a row of zeros under eps 0 has no norm."""
    x = torch.full((5, 384), 2.0 ** 120, dtype=torch.bfloat16, device="cuda")
    x[0, 5], x[1, 5], x[2], x[3], x[3, 7] = float("nan"), float("inf"), 0.0, 2.0 ** -120, float("inf")
    q, scales = norm_codes(x, eps=0.0)
    nan = torch.isnan(q.float() * scales.repeat_interleave(128, 1)).cpu()
    assert bool(nan[0].all()) and bool(nan[2].all()) and not bool(nan[4].any())
    for row, at in ((1, 5), (3, 7)):
        assert nan[row].nonzero().flatten().tolist() == [at]
        assert not bool(q[row, 128:].float().any())
