"""A status read of some bits takes those and leaves the others."""
import pytest
import torch

pytestmark = pytest.mark.gpu

k = pytest.importorskip("krea2_hrx_b200")
from krea2_hrx_b200 import ops, parallel  # noqa: E402
from krea2_hrx_b200._lib import check, lib  # noqa: E402


def test_bits_are_taken_by_their_mask():
    """The bit is raised by a bounded wait on a slot that nothing sets, which gives up after two seconds."""
    # a product and a cross attention, so that their words are read as well
    codes, scale = torch.zeros((4, 128), dtype=torch.float8_e4m3fn, device="cuda"), torch.ones((4, 1), device="cuda")
    ops.gemm_fp8_128(codes, scale, codes, scale[:1], torch.empty((4, 4), dtype=torch.bfloat16, device="cuda"))
    q = torch.zeros((1, 4, 2, 64), dtype=torch.bfloat16, device="cuda")
    ops.cross_attention(q, q, q, torch.empty_like(q))
    assert k.device_status() == 0
    flags = torch.zeros(8, dtype=torch.int32, device="cuda")
    flags[0] = 1
    check(lib().krea2_shard_wait(torch.cuda.current_stream().cuda_stream, flags.data_ptr(), 2, 1, None))
    assert k.device_status(15 | 32 | 64 | 128) == 0
    assert k.device_status(0) == 0
    with pytest.raises(k.Runtime, match="device status 16"):
        parallel.require_clean_status()
    assert k.device_status() == 0
