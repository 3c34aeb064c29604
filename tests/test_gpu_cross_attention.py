"""Cross attention against its definition in 64 bits: lengths, masks, head layouts, pitches, what lies in keys that do not
count; and a cross-attention sublayer of all the operators together."""
import math
import os
import subprocess
import sys

import pytest
import torch

import operator_definitions as defs
from operator_definitions import KINDS

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

k = pytest.importorskip("krea2_hrx_b200")
from krea2_hrx_b200 import ops  # noqa: E402


def rows_of(batch, length, heads, dim, dtype, seed, spare=0, scale=1.0):
    buffer = torch.full((batch, length, heads * dim + spare), 3.0, dtype=dtype, device="cuda")
    buffer[..., : heads * dim] = (torch.randn((batch, length, heads * dim), generator=torch.Generator().manual_seed(seed)) * scale).cuda().to(dtype)
    return buffer[..., : heads * dim].view(batch, length, heads, dim)


def attend(batch, q_len, kv_len, q_heads, kv_heads, dim, dtype, lengths=None, mask=None, spare=0, scale=None, spread=1.0, poison=True):
    q, key = rows_of(batch, q_len, q_heads, dim, dtype, 1, spare, spread), rows_of(batch, kv_len, kv_heads, dim, dtype, 2, 2 * spare, spread)
    value = rows_of(batch, kv_len, kv_heads, dim, dtype, 3, spare)
    lengths = None if lengths is None else torch.tensor(lengths, dtype=torch.int32)
    if poison:  # keys that do not count hold whatever a padded batch leaves there
        for b in range(batch):
            skip = torch.zeros(kv_len, dtype=torch.bool)
            if lengths is not None:
                skip[max(0, int(lengths[b])):] = True
            if mask is not None:
                skip |= mask[b] == 0
            key[b, skip.cuda()], value[b, skip.cuda()] = float("nan"), float("inf")
    guard = torch.full((batch, q_len + 1, q_heads * dim + spare), 7.0, dtype=dtype, device="cuda")
    out = guard[:, :q_len, : q_heads * dim].view(batch, q_len, q_heads, dim) if not spare else guard[:, :q_len, : q_heads * dim].unflatten(-1, (q_heads, dim))
    ops.cross_attention(q, key, value, out, kv_lengths=None if lengths is None else lengths.cuda(), key_mask=None if mask is None else mask.cuda(), scale=scale)
    torch.cuda.synchronize()
    defs.check_cross(out, q, key, value, dim ** -0.5 if scale is None else scale, lengths, mask)
    assert bool((guard[:, q_len] == 7.0).all()) and bool((guard[..., q_heads * dim:] == 7.0).all()), "what lies beside the output is left as it was"
    assert k.device_status() == 0


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("batch,q_len,kv_len,q_heads,kv_heads,dim", [
    (1, 1, 1, 1, 1, 64), (1, 1, 512, 48, 12, 128), (2, 1, 77, 8, 2, 128), (3, 7, 127, 4, 4, 64), (1, 128, 128, 2, 2, 128), (1, 129, 129, 3, 1, 128),
    (2, 33, 256, 6, 2, 64), (1, 300, 257, 4, 1, 80), (2, 65, 1000, 2, 1, 40), (1, 5, 4109, 2, 2, 64), (4, 2, 300, 5, 1, 8), (1, 1000, 40, 12, 3, 120),
    (1, 513, 640, 2, 2, 128), (1, 700, 384, 3, 3, 64), (7, 1, 2050, 7, 1, 96), (1, 40, 1, 16, 4, 128), (1, 3, 9000, 1, 1, 128)])
def test_cross_attention(kind, batch, q_len, kv_len, q_heads, kv_heads, dim):
    attend(batch, q_len, kv_len, q_heads, kv_heads, dim, KINDS[kind])


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("q_len,dim,spare", [(1, 128, 0), (9, 64, 8), (150, 128, 64), (260, 72, 0)])
def test_lengths(kind, q_len, dim, spare):
    """Empty, one key, ends inside, at and just past tiles, more than there are, fewer than none; rows with a pitch."""
    attend(9, q_len, 300, 4, 2, dim, KINDS[kind], lengths=[0, 1, 127, 128, 129, 299, 300, 1000, -5], spare=spare)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("q_len,kv_len,dim", [(1, 200, 128), (5, 1, 64), (140, 700, 64), (300, 513, 128)])
def test_masks(kind, q_len, kv_len, dim):
    g = torch.Generator().manual_seed(7)
    mask = torch.rand((5, kv_len), generator=g) < 0.7
    mask[1] = False
    mask[2] = False
    mask[2, kv_len - 1] = True
    mask[3, : kv_len // 2] = False
    attend(5, q_len, kv_len, 4, 2, dim, KINDS[kind], mask=mask)
    attend(5, q_len, kv_len, 4, 2, dim, KINDS[kind], mask=mask.to(torch.uint8) * 3, lengths=[kv_len, kv_len // 2, kv_len, kv_len // 2, kv_len // 3 + 1])


def test_large_scores_and_another_scale():
    """Scores in the hundreds: nearly one-hot rows whose maximum moves from tile to tile."""
    attend(1, 200, 700, 2, 1, 128, torch.bfloat16, spread=5.0, scale=0.3)
    attend(1, 3, 700, 2, 1, 64, torch.float16, spread=4.0, scale=1.0)
    # growing keys: every tile raises the maximum
    q, key, value = rows_of(1, 130, 1, 64, torch.bfloat16, 1), rows_of(1, 600, 1, 64, torch.bfloat16, 2), rows_of(1, 600, 1, 64, torch.bfloat16, 3)
    q[:] = q.abs()
    key[:] = key.abs() * torch.linspace(0.1, 3.0, 600, device="cuda")[None, :, None, None]
    out = torch.empty_like(q)
    ops.cross_attention(q, key, value, out)
    defs.check_cross(out, q, key, value, 0.125)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("q_len,kv_len", [(1, 16384), (1000, 4096)])
def test_many_small_weights_count(kind, q_len, kv_len):
    """One key takes nearly all of a row, the others 2^-26 of it each and carry the only values: rounded on their own for the
    second product, they must not vanish."""
    dtype = KINDS[kind]
    q, key = torch.zeros((1, q_len, 2, 64), dtype=dtype, device="cuda"), torch.zeros((1, kv_len, 2, 64), dtype=dtype, device="cuda")
    q[..., 0], key[:, 1:, :, 0], value = 1.0, -26.0, torch.ones_like(key)
    value[:, 0] = 0.0
    out = torch.empty_like(q)
    ops.cross_attention(q, key, value, out, scale=math.log(2.0))
    small = (kv_len - 1) * 2.0 ** -26
    # 2^-26 is a power of two, which a weight that is off by its f32 arguments' rounding (26 * 2^-23 at most) rounds to; the
    # output is rounded once.
    want, eps = small / (1.0 + small), torch.finfo(dtype).eps / 2
    assert float((out.double() - want).abs().max()) <= want * (eps + 1e-5)


def test_no_keys_at_all():
    q = rows_of(2, 5, 4, 64, torch.bfloat16, 1)
    empty, out = torch.empty((2, 0, 2, 64), dtype=torch.bfloat16, device="cuda"), torch.full_like(q, 9.0)
    ops.cross_attention(q, empty, empty, out)
    assert not bool(out.float().any())


def test_nan_in_a_counting_key_is_not_hidden():
    q, key, value = rows_of(1, 140, 2, 64, torch.float16, 1), rows_of(1, 200, 2, 64, torch.float16, 2), rows_of(1, 200, 2, 64, torch.float16, 3)
    key[0, 150, 0, 3] = float("nan")
    out = torch.empty_like(q)
    ops.cross_attention(q, key, value, out)
    assert bool(torch.isnan(out[0, :, 0]).all()) and not bool(torch.isnan(out[0, :, 1]).any())


@pytest.mark.parametrize("q_len", [1, 200])
def test_views_of_wider_tensors_and_shared_states(q_len):
    """q out of a q|k|v row, k and v out of one k|v row, the same encoder states for every item of a batch."""
    fused = rows_of(3, q_len, 12, 64, torch.bfloat16, 1)
    q = fused[:, :, 2:6]
    kv = rows_of(1, 150, 8, 64, torch.bfloat16, 2).expand(3, 150, 8, 64)
    key, value = kv[:, :, :2], kv[:, :, 4:6]
    out = torch.empty((3, q_len, 4, 64), dtype=torch.bfloat16, device="cuda")
    ops.cross_attention(q, key, value, out)
    defs.check_cross(out, q, key, value, 0.125)


@pytest.mark.parametrize("q_len", [1, 150])
def test_sequence_first_layouts_and_a_shared_mask(q_len):
    """[length][batch][heads][dim] tensors seen batch first, outputs too; one mask for the whole batch, one query for all."""
    q, key, value = (rows_of(n, 3, h, 64, torch.float16, n).transpose(0, 1) for n, h in ((q_len, 4), (300, 2), (301, 2)))
    value = value[:, :300]
    out = torch.full((q_len + 1, 3, 4, 64), 7.0, dtype=torch.float16, device="cuda")
    mask = (torch.rand(300, generator=torch.Generator().manual_seed(1)) < 0.5).expand(3, 300)
    ops.cross_attention(q, key, value, out[:q_len].transpose(0, 1), key_mask=mask.cuda()[:1].expand(3, 300))
    defs.check_cross(out[:q_len].transpose(0, 1), q, key, value, 0.125, key_mask=mask)
    assert bool((out[q_len] == 7.0).all())
    shared = q[:1].expand(3, q_len, 4, 64)
    again = torch.empty((3, q_len, 4, 64), dtype=torch.float16, device="cuda")
    ops.cross_attention(shared, key, value, again)
    defs.check_cross(again, shared, key, value, 0.125)


@pytest.mark.parametrize("heads", [3, 5, 7, 24, 128])
def test_heads_that_do_not_fill_a_tile(heads):
    """Row tiles of 128 // heads queries: the rows left over in a tile belong to nobody."""
    attend(2, 100, 200, heads, 1, 64, torch.bfloat16, lengths=[200, 77])


def test_first_calls_inside_a_capture(tmp_path):
    """A process whose first call of every operator is recorded into a graph."""
    script = tmp_path / "capture.py"
    script.write_text(f"""
import sys
sys.path[:0] = [{ROOT!r}, {os.path.join(ROOT, 'tests')!r}]
import torch
import operator_definitions as defs
from krea2_hrx_b200 import ops
g = torch.Generator().manual_seed(0)
t = lambda *shape: torch.randn(shape, generator=g).to(torch.bfloat16).cuda()
codes = lambda m, k: torch.empty((m, k), dtype=torch.float8_e4m3fn, device="cuda")
x, w, out = t(300, 512), t(384, 512), torch.empty((300, 384), dtype=torch.bfloat16, device="cuda")
a, a_scale, b, b_scale = codes(300, 512), torch.empty((300, 4), device="cuda"), codes(384, 512), torch.ones((3, 4), device="cuda")
b.view(torch.uint8).copy_(w.to(torch.float8_e4m3fn).view(torch.uint8))
small = torch.empty((5, 384), dtype=torch.bfloat16, device="cuda")
q, kv, o = t(2, 50, 4, 64), t(2, 70, 2, 64), torch.empty((2, 50, 4, 64), dtype=torch.bfloat16, device="cuda")
f, _ = ops.rotary_frequencies(64)
r = torch.empty((100, 4, 64), dtype=torch.bfloat16, device="cuda")
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    ops.prepare_norm_fp8(x, None, a, a_scale, weight_offset=1.0)
    ops.gemm_fp8_128(a, a_scale, b, b_scale, out)
    ops.gemm_fp8_128(a[:5], a_scale[:5], b, b_scale, small)
    ops.rotary(q.view(100, 4, 64), None, r, None, f)
    ops.cross_attention(q, kv, kv, o)
graph.replay()
torch.cuda.synchronize()
defs.check_codes(a, a_scale, defs.norm_rows(x, None, None, 1e-5, 1.0)[0], 60)
defs.check_product(out, a, a_scale, b, b_scale)
defs.check_product(small, a.view(torch.uint8)[:5].view(a.dtype), a_scale[:5], b, b_scale)
defs.check_rotary(r, q.view(100, 4, 64), torch.arange(100), f, 1.0, "interleaved", False)
defs.check_cross(o, q, kv, kv, 0.125)
print("captured")
""")
    done = subprocess.run([sys.executable, str(script)], capture_output=True, text=True, timeout=300)
    assert done.returncode == 0 and "captured" in done.stdout, done.stdout + done.stderr


@pytest.mark.parametrize("q_len", [2, 300])
def test_captured_and_replayed_beside_another(q_len):
    sets = [[rows_of(2, n, h, 64, torch.bfloat16, s + i) for i, (n, h) in enumerate(((q_len, 4), (700, 2), (700, 2)))] for s in (0, 10)]
    lengths = [torch.tensor([700, 5], dtype=torch.int32, device="cuda") for _ in sets]
    outs = [torch.empty_like(s[0]) for s in sets]
    for s, n, out in zip(sets, lengths, outs):
        ops.cross_attention(*s, out, kv_lengths=n)
    torch.cuda.synchronize()
    graphs, streams = [], [torch.cuda.Stream() for _ in sets]
    for s, n, out, stream in zip(sets, lengths, outs, streams):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            ops.cross_attention(*s, out, kv_lengths=n)
        graphs.append(graph)
    lengths[0].copy_(torch.tensor([300, 0], dtype=torch.int32))
    sets[1][2].mul_(2.0)
    torch.cuda.synchronize()
    for _ in range(3):
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
    torch.cuda.synchronize()
    for s, n, out in zip(sets, lengths, outs):
        defs.check_cross(out, *s, 0.125, n.cpu())
    first = outs[0].clone()
    for _ in range(10):
        graphs[0].replay()
        torch.cuda.synchronize()
        assert torch.equal(first, outs[0]), "the same inputs give the same bits"


def test_refusals():
    q, key = torch.zeros((2, 3, 4, 64), dtype=torch.bfloat16, device="cuda"), torch.zeros((2, 5, 2, 64), dtype=torch.bfloat16, device="cuda")
    n, mask = torch.ones(2, dtype=torch.int32, device="cuda"), torch.ones((2, 5), dtype=torch.bool, device="cuda")
    for call in (lambda: ops.cross_attention(q, key, key[:, :4], q), lambda: ops.cross_attention(q, key, key, q[:, :2]),
                 lambda: ops.cross_attention(q.float(), key.float(), key.float(), q.float()), lambda: ops.cross_attention(q, key.half(), key.half(), q),
                 lambda: ops.cross_attention(q, key, key, q, kv_lengths=n.long()), lambda: ops.cross_attention(q, key, key, q, kv_lengths=n[:1]),
                 lambda: ops.cross_attention(q, key, key, q, key_mask=mask[:, :4]), lambda: ops.cross_attention(q, key, key, q, key_mask=mask.float()),
                 lambda: ops.cross_attention(q, key[..., :32], key[..., :32], q), lambda: ops.cross_attention(q[:, :, :3], key, key, q[:, :, :3].clone()),
                 lambda: ops.cross_attention(q, key, key, q.clone(), scale=-1.0), lambda: ops.cross_attention(q[:, :0], key, key, q[:, :0]),
                 lambda: ops.cross_attention(q.cpu(), key, key, q)):
        with pytest.raises(k.InvalidArgument):
            call()


def test_a_cross_attention_sublayer():
    """residual + norm -> e4m3 query projection -> rotary -> cross attention to projected encoder states -> e4m3 output
    projection -> residual + norm; every step against its definition on what the step before it left."""
    dtype, width, states, q_heads, kv_heads, dim, batch, q_len, kv_len = torch.bfloat16, 512, 320, 8, 2, 64, 2, 75, 90
    g = torch.Generator().manual_seed(0)
    layer = lambda n, m: ops.QuantizedFp8((torch.randn((n, m), generator=g) * m ** -0.5).cuda())  # noqa: E731
    to_q, to_kv, to_out = layer(q_heads * dim, width), layer(2 * kv_heads * dim, states), layer(width, q_heads * dim)
    norm = (torch.randn(width, generator=g) * 0.1).cuda()
    x, delta = (torch.randn((batch * q_len, width), generator=g).cuda().to(dtype) for _ in range(2))
    encoded = torch.randn((batch * kv_len, states), generator=g).cuda().to(dtype)
    lengths = torch.tensor([90, 31], dtype=torch.int32, device="cuda")
    frequencies, magnitude = ops.rotary_frequencies(dim)
    positions = {n: torch.arange(n, dtype=torch.int32, device="cuda").repeat(batch) for n in (q_len, kv_len)}

    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        codes, total = to_q.buffers(batch * q_len), torch.empty_like(x)
        q = to_q.forward_norm(x, norm, residual=delta, sum_out=total, weight_offset=1.0, buffers=codes).view(-1, q_heads, dim)
        kv_codes = to_kv.buffers(batch * kv_len)
        kv = to_kv.forward(encoded, buffers=kv_codes).view(-1, 2 * kv_heads, dim)
        turned, keys = torch.empty_like(q), torch.empty((batch * kv_len, kv_heads, dim), dtype=dtype, device="cuda")
        ops.rotary(q, None, turned, None, frequencies, positions=positions[q_len], layout="half")
        ops.rotary(kv[:, :kv_heads], None, keys, None, frequencies, positions=positions[kv_len], layout="half")
        out = torch.empty((batch, q_len, q_heads, dim), dtype=dtype, device="cuda")
        values = kv.view(batch, kv_len, 2 * kv_heads, dim)[:, :, kv_heads:]
        ops.cross_attention(turned.view(out.shape), keys.view(batch, kv_len, kv_heads, dim), values, out, kv_lengths=lengths)
        out_codes = to_out.buffers(batch * q_len)
        update = to_out.forward(out.view(batch * q_len, -1), buffers=out_codes)
        last, last_sum = to_q.buffers(batch * q_len), torch.empty_like(x)
        ops.prepare_norm_fp8(update, norm, *last, residual=total, sum_out=last_sum, weight_offset=1.0)
    stream.synchronize()

    want, want_sum = defs.norm_rows(x, delta, norm, 1e-5, 1.0)
    assert torch.equal(total.cpu(), want_sum)
    defs.check_codes(*codes, want, 60)
    defs.check_product(q.view(-1, q_heads * dim), *codes, to_q.weight, to_q.scales)
    defs.check_codes(*kv_codes, defs.f64(encoded), 0)
    defs.check_product(kv.view(batch * kv_len, -1), *kv_codes, to_kv.weight, to_kv.scales)
    defs.check_rotary(turned, q, positions[q_len].cpu(), frequencies, magnitude, "half", False)
    defs.check_rotary(keys, kv[:, :kv_heads], positions[kv_len].cpu(), frequencies, magnitude, "half", False)
    defs.check_cross(out, turned.view(out.shape), keys.view(batch, kv_len, kv_heads, dim), values, dim ** -0.5, lengths.cpu())
    defs.check_codes(*out_codes, defs.f64(out.view(batch * q_len, -1)), 0)
    defs.check_product(update, *out_codes, to_out.weight, to_out.scales)
    want, want_sum = defs.norm_rows(update, total, norm, 1e-5, 1.0)
    assert torch.equal(last_sum.cpu(), want_sum)
    defs.check_codes(*last, want, 60)
    assert k.device_status() == 0
