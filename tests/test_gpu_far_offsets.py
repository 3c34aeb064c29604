"""The e4m3, rotary and cross-attention operators on tensors whose rows lie more than 2^32 elements apart."""
import pytest
import torch

import operator_definitions as defs

pytestmark = pytest.mark.gpu

k = pytest.importorskip("krea2_hrx_b200")
from krea2_hrx_b200 import ops  # noqa: E402

FAR = 2 ** 32 + 64


@pytest.fixture(scope="module")
def store():
    """Two stretches of 8.6 GB, one to read from and one to write to."""
    if torch.cuda.mem_get_info()[0] < 24e9:
        pytest.skip("needs 18 GB of free device memory")
    pair = [torch.empty(FAR + 2 ** 20, dtype=torch.bfloat16, device="cuda") for _ in range(2)]
    yield pair
    pair.clear()
    torch.cuda.empty_cache()


def far_rows(buffer, values):
    """`values` [2][...] as a view whose second item lies FAR elements behind the first."""
    view = buffer.as_strided(values.shape, (FAR, *values.stride()[1:]))
    view.copy_(values)
    return view


def seeded(*shape):
    return torch.randn(shape, generator=torch.Generator().manual_seed(1)).cuda().to(torch.bfloat16)


def test_codes_and_product(store):
    x = far_rows(store[0], seeded(2, 320))
    codes = store[1].view(torch.float8_e4m3fn).as_strided((2, 320), (FAR, 1))
    scales, total = torch.empty((2, 3), device="cuda"), store[1][2 ** 19:].as_strided((2, 320), (FAR, 1))
    ops.prepare_norm_fp8(x, None, codes, scales, residual=x, sum_out=total, weight_offset=1.0)
    want, want_sum = defs.norm_rows(x, x, None, 1e-5, 1.0)
    assert torch.equal(total.cpu(), want_sum)
    defs.check_codes(codes.view(torch.uint8).contiguous().view(codes.dtype), scales, want, 60)
    w, w_scale = ops.QuantizedFp8(seeded(200, 320)).weight, torch.rand((2, 3), device="cuda")
    for c in (store[0].as_strided((2, 200), (FAR, 1)), torch.empty((2, 200), dtype=torch.bfloat16, device="cuda")):
        ops.gemm_fp8_128(codes, scales, w, w_scale, c)
        defs.check_product(c, codes.view(torch.uint8).contiguous().view(codes.dtype), scales, w, w_scale)
    # many rows of a: the last ones' outputs lie behind 2^31 elements
    rows = 16380
    a, a_scale = ops.QuantizedFp8(seeded(rows, 320)).weight, torch.rand((rows, 3), device="cuda")
    c = store[0].as_strided((rows, 200), (2 ** 18 + 8, 1))
    ops.gemm_fp8_128(a, a_scale, w, w_scale, c)
    last = slice(rows - 40, rows)
    defs.check_product(c[last], a.view(torch.uint8)[last].view(a.dtype), a_scale[last], w, w_scale)


@pytest.mark.parametrize("layout,rotary_dim", [("interleaved", 64), ("half", 64), ("half", 34)])
def test_rotary(store, layout, rotary_dim):
    q = far_rows(store[0], seeded(2, 3, 64))
    out = store[1].as_strided((2, 3, 64), (FAR, 64, 1))
    frequencies, _ = ops.rotary_frequencies(rotary_dim)
    ops.rotary(q, None, out, None, frequencies, layout=layout)
    defs.check_rotary(out, q, torch.arange(2), frequencies, 1.0, layout, False)


@pytest.mark.parametrize("q_len", [1, 200])
def test_cross_attention(store, q_len):
    q, key, value = seeded(2, q_len, 2, 64), seeded(2, 300, 1, 64), seeded(2, 300, 1, 64) + 1.0
    q, key, value = (far_rows(store[0][at:], t) for at, t in ((0, q), (2 ** 17, key), (2 ** 18, value)))
    out = store[1].as_strided((2, q_len, 2, 64), (FAR, 128, 64, 1))
    ops.cross_attention(q, key, value, out)
    defs.check_cross(out, q, key, value, 0.125)
