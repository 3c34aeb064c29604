"""Tensors without channels, heads or rows are refused by name, whatever the wrapper computes from their shape on the way."""
import pytest
import torch

import krea2_hrx_b200 as k
from krea2_hrx_b200 import ops

E4M3 = torch.float8_e4m3fn


def zeros(*shape, d=torch.bfloat16):
    return torch.zeros(shape).to(d)


CALLS = [
    lambda z: ops.cross_attention(z(1, 2, 2, 0), z(1, 3, 2, 0), z(1, 3, 2, 0), z(1, 2, 2, 0)),
    lambda z: ops.cross_attention(z(1, 2, 0, 64), z(1, 3, 0, 64), z(1, 3, 0, 64), z(1, 2, 0, 64)),
    lambda z: ops.cross_attention(z(0, 2, 2, 64), z(0, 3, 2, 64), z(0, 3, 2, 64), z(0, 2, 2, 64)),
    lambda z: ops.rotary(z(3, 2, 0), None, z(3, 2, 0), None, z(0, d=torch.float64)),
    lambda z: ops.rotary(z(3, 0, 64), None, z(3, 0, 64), None, z(32, d=torch.float64)),
    lambda z: ops.rotary(z(0, 2, 64), z(0, 2, 64), z(0, 2, 64), z(0, 2, 64), z(32, d=torch.float64)),
    lambda z: ops.prepare_plain_fp8(z(3, 0), z(3, 0, d=E4M3), z(3, 0, d=torch.float32)),
    lambda z: ops.prepare_norm_fp8(z(0, 128), None, z(0, 128, d=E4M3), z(0, 1, d=torch.float32), residual=z(0, 128), sum_out=z(0, 128)),
    lambda z: ops.gemm_fp8_128(z(3, 0, d=E4M3), z(3, 0, d=torch.float32), z(4, 0, d=E4M3), z(1, 0, d=torch.float32), z(3, 4)),
    lambda z: ops.gemm_fp8_128(z(3, 128, d=E4M3), z(3, 1, d=torch.float32), z(0, 128, d=E4M3), z(0, 1, d=torch.float32), z(3, 0)),
]


@pytest.mark.parametrize("call", CALLS)
def test_empty_tensors_are_refused(call):
    with pytest.raises(k.InvalidArgument):
        call(zeros)


@pytest.mark.gpu
@pytest.mark.parametrize("call", CALLS)
def test_empty_tensors_are_refused_on_the_device(call):
    with pytest.raises(k.InvalidArgument):
        call(lambda *shape, d=torch.bfloat16: zeros(*shape, d=d).cuda())
