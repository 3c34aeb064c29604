"""Rotary positions against their definition in 64 bits, forwards and backwards."""
import pytest
import torch

import operator_definitions as defs
from operator_definitions import KINDS

pytestmark = pytest.mark.gpu

k = pytest.importorskip("krea2_hrx_b200")
from krea2_hrx_b200 import ops  # noqa: E402


def heads(tokens, count, dim, dtype, seed, pitch=None):
    """[tokens][count][dim] inside rows of that pitch."""
    buffer = torch.full((tokens + 1, pitch or count * dim), 5.0, dtype=dtype, device="cuda")
    buffer[:tokens, : count * dim] = torch.randn((tokens, count * dim), generator=torch.Generator().manual_seed(seed)).cuda().to(dtype)
    return buffer, buffer[:tokens, : count * dim].view(tokens, count, dim)


CASES = [  # tokens, q heads, kv heads, head_dim, rotary_dim, spare elements of a row
    (1, 48, 12, 128, 128, 0), (5, 3, 1, 64, 64, 8), (7, 4, 4, 64, 32, 0), (3, 2, 2, 128, 96, 40), (130, 8, 2, 80, 80, 0), (2, 5, 1, 80, 20, 4),
    (4, 1, 1, 2, 2, 0), (9, 3, 3, 66, 34, 1), (17, 2, 1, 256, 128, 0), (33, 1, 1, 512, 512, 0), (6, 2, 0, 128, 128, 0), (65, 6, 2, 96, 48, 0),
    (40, 1, 1, 64, 16, 0), (300, 2, 1, 40, 40, 0)]


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("layout", ["interleaved", "half"])
@pytest.mark.parametrize("tokens,q_heads,kv_heads,dim,rotary_dim,spare", CASES)
def test_rotary(kind, layout, tokens, q_heads, kv_heads, dim, rotary_dim, spare):
    dtype = KINDS[kind]
    frequencies, magnitude = ops.rotary_frequencies(rotary_dim, scaling="parts", factor=4.0, trained=2048.0)
    positions = (torch.arange(tokens, dtype=torch.int32) * 37 - 11)
    for inverse in (False, True):
        _, q = heads(tokens, q_heads, dim, dtype, 1, q_heads * dim + spare)
        kv = heads(tokens, kv_heads, dim, dtype, 2, kv_heads * dim + 2 * spare)[1] if kv_heads else None
        q_rows, q_out = heads(tokens, q_heads, dim, dtype, 3, q_heads * dim + spare)
        k_out = torch.empty_like(kv) if kv_heads else None
        beside = q_rows[:, q_heads * dim:].clone(), q_rows[tokens].clone()
        ops.rotary(q, kv, q_out, k_out, frequencies, positions=positions.cuda(), magnitude=magnitude, layout=layout, inverse=inverse)
        torch.cuda.synchronize()
        defs.check_rotary(q_out, q, positions, frequencies, magnitude, layout, inverse)
        if kv_heads:
            defs.check_rotary(k_out, kv, positions, frequencies, magnitude, layout, inverse)
        assert torch.equal(q_rows[:, q_heads * dim:], beside[0]) and torch.equal(q_rows[tokens], beside[1])


@pytest.mark.parametrize("layout", ["interleaved", "half"])
@pytest.mark.parametrize("dim,rotary_dim", [(128, 128), (128, 64), (66, 34)])
def test_in_place_equals_out_of_place(layout, dim, rotary_dim):
    frequencies, _ = ops.rotary_frequencies(rotary_dim)
    q, kv = heads(50, 4, dim, torch.bfloat16, 1)[1], heads(50, 2, dim, torch.bfloat16, 2)[1]
    q_out, k_out = torch.empty_like(q), torch.empty_like(kv)
    ops.rotary(q, kv, q_out, k_out, frequencies, layout=layout)  # positions are the row numbers
    defs.check_rotary(q_out, q, torch.arange(50), frequencies, 1.0, layout, False)
    ops.rotary(q, kv, q, kv, frequencies, layout=layout)
    assert torch.equal(q, q_out) and torch.equal(kv, k_out)


@pytest.mark.parametrize("scaling", ["none", "linear", "base", "parts"])
def test_far_positions(scaling):
    """Up to the ends of int32: an f32 product of position and frequency would be off by whole turns."""
    frequencies, magnitude = ops.rotary_frequencies(64, base=500000.0, scaling=scaling, factor=16.0, trained=8192.0)
    positions = torch.tensor([0, 1, 4095, 131071, 1000003, 16777217, 2147483647, -2147483648, -1], dtype=torch.int32)
    q = heads(len(positions), 2, 64, torch.float16, 4)[1]
    out = torch.empty_like(q)
    ops.rotary(q, None, out, None, frequencies, positions=positions.cuda(), magnitude=magnitude, layout="half")
    defs.check_rotary(out, q, positions, frequencies, magnitude, "half", False)


@pytest.mark.parametrize("layout", ["interleaved", "half"])
def test_inverse_is_the_gradient(layout):
    """<turn(x), g> has the gradient turn_back(g): against the definition's derivative and against differences of it."""
    frequencies, magnitude = ops.rotary_frequencies(24, scaling="parts", factor=4.0, trained=64.0)
    positions = torch.arange(6, dtype=torch.int32) * 5
    x, g = heads(6, 2, 32, torch.float16, 1)[1], heads(6, 2, 32, torch.float16, 2)[1]
    grad = torch.empty_like(g)
    ops.rotary(g, None, grad, None, frequencies, positions=positions.cuda(), magnitude=magnitude, layout=layout, inverse=True)
    defs.check_rotary(grad, g, positions, frequencies, magnitude, layout, True)
    turned = lambda t: (defs.rotary(t, positions, frequencies, magnitude, layout, False)[0] * defs.f64(g)).sum()  # noqa: E731
    for at in [(0, 0, 0), (3, 1, 5), (5, 0, 13), (2, 1, 23), (4, 1, 30)]:
        step = torch.zeros(x.shape, dtype=torch.float64)
        step[at] = 2.0 ** -6
        difference = (turned(defs.f64(x) + step) - turned(defs.f64(x) - step)) / 2.0 ** -5  # linear: exact up to f64
        reach = defs.rotary(g, positions, frequencies, magnitude, layout, True)[1][at]
        assert abs(float(difference) - float(grad[at])) <= 2.0 ** -11 * abs(float(difference)) + 10 * defs.F32 * float(reach) + 1e-10


def test_captured_on_another_stream():
    frequencies, _ = ops.rotary_frequencies(64)
    q = heads(100, 4, 64, torch.bfloat16, 1)[1]
    out = torch.empty_like(q)
    positions = torch.arange(100, dtype=torch.int32, device="cuda")
    ops.rotary(q, None, out, None, frequencies, positions=positions)
    torch.cuda.synchronize()
    graph, stream = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.graph(graph, stream=stream):
        ops.rotary(q, None, out, None, frequencies, positions=positions)
    positions += 9000
    torch.cuda.synchronize()
    graph.replay()
    torch.cuda.synchronize()
    defs.check_rotary(out, q, positions.cpu(), frequencies, 1.0, "interleaved", False)


def test_refusals():
    f = torch.ones(32, dtype=torch.float64, device="cuda")
    q = torch.zeros((3, 2, 64), dtype=torch.bfloat16, device="cuda")
    for call in (lambda: ops.rotary(q, q, q, None, f), lambda: ops.rotary(q, None, q[:2], None, f), lambda: ops.rotary(q.float(), None, q.float(), None, f),
                 lambda: ops.rotary(q, None, q, None, f.float()), lambda: ops.rotary(q, None, q, None, f, layout="other"),
                 lambda: ops.rotary(q, None, q, None, f, positions=torch.zeros(3, dtype=torch.int64, device="cuda")),
                 lambda: ops.rotary(q, None, q, None, f, positions=torch.zeros(2, dtype=torch.int32, device="cuda")),
                 lambda: ops.rotary(q.transpose(0, 1), None, q.transpose(0, 1), None, f), lambda: ops.rotary(q[:, :, :32], None, q[:, :, :32], None, f),
                 lambda: ops.rotary(q, q.half(), q, q.half(), f), lambda: ops.rotary(q, None, q, None, torch.cat([f, f]))):
        with pytest.raises(k.InvalidArgument):
            call()
