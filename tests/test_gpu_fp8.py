"""The e4m3 prologues and product against their definitions in 64 bits, at the sizes, pitches and values where they can go
wrong, and as a projection."""
import math

import pytest
import torch

import operator_definitions as defs
from operator_definitions import KINDS

pytestmark = pytest.mark.gpu

k = pytest.importorskip("krea2_hrx_b200")
from krea2_hrx_b200 import ops  # noqa: E402

E4M3 = torch.float8_e4m3fn


def rows_of(rows, width, dtype, seed, pitch=None, scale=1.0):
    """Seeded rows with large channels, in a buffer of that pitch."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn((rows, width), generator=g) * torch.where(torch.rand(width, generator=g) < 0.02, 20.0, 1.0) * scale
    buffer = torch.zeros((rows, pitch or width), dtype=dtype, device="cuda")
    buffer[:, :width] = x.cuda().to(dtype)
    return buffer[:, :width]


def code_buffers(rows, width, pitch=None):
    """Codes and scales to write, in sentinels: 0x55 beyond the rows' ends and behind the last row."""
    pitch = pitch or -(-width // 16) * 16
    q = torch.full((rows + 1, pitch), 0x55, dtype=torch.uint8, device="cuda")
    return q, q.view(E4M3)[:rows, :width], torch.full((rows + 1, defs.groups(width)), -7.0, device="cuda")


def check_untouched(q, scales, rows, width):
    assert bool((q[:rows, width:] == 0x55).all()) and bool((q[rows] == 0x55).all()) and bool((scales[rows] == -7.0).all())


NORM_ROUNDINGS = 60  # 32 sequential and 10 tree additions of the squares (halved by the root), the root's and factor's


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("rows,width,extra", [(1, 6144, 0), (3, 1, 0), (2, 127, 0), (5, 128, 0), (4, 129, 8), (33, 1000, 24), (7, 2056, 0), (3, 8192, 64),
                                              (2, 16384, 0), (2, 12345, 3), (2, 32768, 0), (700, 320, 0)])
def test_norm_codes(kind, rows, width, extra):
    dtype = KINDS[kind]
    x, residual = rows_of(rows, width, dtype, 1, width + extra), rows_of(rows, width, dtype, 2, width + 2 * extra, 3.0)
    weight = (torch.randn(width, generator=torch.Generator().manual_seed(3)) * 0.1).cuda()
    for case in ("bare", "weight", "sum", "in place"):
        q, view, scales = code_buffers(rows, width)
        source, second = x.clone() if case == "in place" else x, residual if case in ("sum", "in place") else None
        target = source if case == "in place" else torch.full_like(x, 9.0) if case == "sum" else None
        want, total = defs.norm_rows(source, second, weight if case != "bare" else None, 1e-5, 1.0)
        ops.prepare_norm_fp8(source, weight if case != "bare" else None, view, scales[:rows], residual=second, sum_out=target, weight_offset=1.0)
        torch.cuda.synchronize()
        defs.check_codes(view, scales[:rows], want, NORM_ROUNDINGS)
        check_untouched(q, scales, rows, width)
        if total is not None:
            assert torch.equal(target.cpu(), total)
    assert k.device_status() == 0


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("rows,width,extra", [(1, 16384, 0), (1043, 256, 0), (3, 129, 0), (2, 1, 7), (9, 2880, 16), (2, 32768, 8)])
def test_plain_codes(kind, rows, width, extra):
    x = rows_of(rows, width, KINDS[kind], 4, width + extra)
    q, view, scales = code_buffers(rows, width, pitch=-(-width // 16) * 16 + 32)
    ops.prepare_plain_fp8(x, view, scales[:rows])
    torch.cuda.synchronize()
    defs.check_codes(view, scales[:rows], defs.f64(x), 0)
    check_untouched(q, scales, rows, width)


def test_rows_of_zeros_tiny_and_largest_values():
    x = torch.zeros((6, 256), dtype=torch.bfloat16, device="cuda")
    x[1] = 2.0 ** -130
    x[2] = 3.0e38
    x[3, :128] = 1e-30
    x[4, 200] = -1.0
    q, view, scales = code_buffers(6, 256)
    ops.prepare_plain_fp8(x, view, scales[:6])
    torch.cuda.synchronize()
    assert bool((scales[0] == 2.0 ** -126).all()) and not bool(view[0].float().any())
    assert bool((view[2].float() == 448.0).all()) and float(view[4].float()[200]) == -448.0
    # the exact quotient of a tiny row by the floored scale is below half of the smallest code
    defs.check_codes(view, scales[:6], defs.f64(x), 0)
    ops.prepare_norm_fp8(x, None, view, scales[:6], eps=0.0 + 1e-12, weight_offset=1.0)
    assert not bool(view[0].float().any())


@pytest.mark.parametrize("norm", [False, True])
def test_nan_and_infinity_stay_where_the_text_says(norm):
    x = torch.ones((3, 384), dtype=torch.float16, device="cuda")
    x[0, 130], x[1, 5] = float("nan"), float("inf")
    _, view, scales = code_buffers(3, 384)
    if norm:
        ops.prepare_norm_fp8(x, None, view, scales[:3], weight_offset=1.0)
    else:
        ops.prepare_plain_fp8(x, view, scales[:3])
    values = view.float() * scales[:3].repeat_interleave(128, 1)
    nan = torch.isnan(values).cpu()
    if norm:  # a NaN reaches the whole row through the mean, an infinity leaves zeros beside itself
        assert bool(nan[0].all()) and nan[1].nonzero().flatten().tolist() == [5]
    else:
        assert nan[0].nonzero().flatten().tolist() == [130] and nan[1].nonzero().flatten().tolist() == list(range(128))
    assert not bool(nan[2].any())


# ------------------------------------------------------------------ product
def operands(m, n, width, seed, a_pitch=None, w_pitch=None):
    """Seeded codes over the whole range under scales of several magnitudes, NaN codes in the padding of the rows."""
    g = torch.Generator().manual_seed(seed)

    def codes(rows, pitch):
        buffer = torch.full((rows, pitch), 0x7f, dtype=torch.uint8)
        buffer[:, :width] = (torch.randn((rows, width), generator=g) * 60).clamp(-448, 448).to(E4M3).view(torch.uint8)
        return buffer.cuda().view(E4M3)[:, :width]

    pitch = -(-width // 16) * 16
    a, w = codes(m, a_pitch or pitch), codes(n, w_pitch or pitch)
    a_scale = torch.exp2(torch.randint(-12, -5, (m, defs.groups(width)), generator=g).float()) * (1 + torch.rand((m, defs.groups(width)), generator=g))
    w_scale = torch.exp2(torch.randint(-12, -7, (defs.groups(n), defs.groups(width)), generator=g).float()) * 1.37
    return a, a_scale.cuda(), w, w_scale.cuda()


SMALL = [(1, 1, 1), (1, 128, 128), (2, 257, 130), (15, 64, 640), (16, 129, 127), (17, 200, 1000), (31, 384, 2048), (33, 8, 4096), (64, 130, 272),
         (65, 1000, 384), (127, 128, 128), (128, 512, 1536), (129, 257, 513)]
LARGE = [(257, 320, 700), (300, 1048, 1024), (513, 513, 129), (1043, 768, 400), (2000, 2056, 256)]


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("m,n,width", SMALL + LARGE)
def test_product(kind, m, n, width):
    a, a_scale, w, w_scale = operands(m, n, width, m * 7 + n)
    c = torch.full((m + 1, n + 3), 77.0, dtype=KINDS[kind], device="cuda")
    ops.gemm_fp8_128(a, a_scale, w, w_scale, c[:m, :n])
    torch.cuda.synchronize()
    defs.check_product(c[:m, :n], a, a_scale, w, w_scale)
    assert bool((c[m] == 77.0).all()) and bool((c[:, n:] == 77.0).all()), "what lies beside the output is left as it was"
    assert k.device_status() == 0


@pytest.mark.parametrize("m,n,width", [(1, 6144, 6144), (8, 6144, 16384), (275, 1024, 16384), (600, 4096, 6144)])
def test_product_at_the_session_s_widths(m, n, width):
    a, a_scale, w, w_scale = operands(m, n, width, 5, w_pitch=width + 64)
    c = torch.empty((m, n), dtype=torch.bfloat16, device="cuda")
    ops.gemm_fp8_128(a, a_scale, w, w_scale, c)
    torch.cuda.synchronize()
    defs.check_product(c, a, a_scale, w, w_scale)


@pytest.mark.parametrize("m,n", [(3, 300), (400, 640)])
def test_product_with_pitches_and_a_lone_special_value(m, n):
    width = 500
    a, a_scale, w, w_scale = operands(m, n, width, 9, a_pitch=1024, w_pitch=560)
    a_scale[1, 2] = float("inf")
    c = torch.zeros((m, n), dtype=torch.float16, device="cuda")
    ops.gemm_fp8_128(a, a_scale, w, w_scale, c)
    torch.cuda.synchronize()
    keep = torch.arange(m) != 1
    keep = keep.cuda()
    defs.check_product(c[keep], a.view(torch.uint8)[keep].view(E4M3), a_scale[keep], w, w_scale)
    assert not bool(torch.isfinite(c[1]).any()), "an infinite scale reaches its row and no other"


@pytest.mark.parametrize("m,n,width", [(5, 512, 4096), (700, 1280, 640)])
def test_product_is_the_same_every_time(m, n, width):
    a, a_scale, w, w_scale = operands(m, n, width, 11)
    first, again = (torch.empty((m, n), dtype=torch.bfloat16, device="cuda") for _ in range(2))
    ops.gemm_fp8_128(a, a_scale, w, w_scale, first)
    for _ in range(20):
        again.fill_(3.0)
        ops.gemm_fp8_128(a, a_scale, w, w_scale, again)
        assert torch.equal(first.view(torch.int16), again.view(torch.int16))


@pytest.mark.parametrize("m", [2, 300])
def test_product_captured_and_replayed_beside_another(m):
    """Two graphs on two streams, replayed at the same time with new inputs."""
    cases, graphs = [operands(m, 640, 1100, s) for s in (1, 2)], []
    outs = [torch.empty((m, 640), dtype=torch.bfloat16, device="cuda") for _ in cases]
    streams = [torch.cuda.Stream() for _ in cases]
    for case, out in zip(cases, outs):
        ops.gemm_fp8_128(*case, out)
    torch.cuda.synchronize()
    for case, out, stream in zip(cases, outs, streams):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            ops.gemm_fp8_128(*case, out)
        graphs.append(graph)
    other = [operands(m, 640, 1100, s) for s in (3, 4)]
    for case, new in zip(cases, other):
        for t, u in zip(case, new):
            (t.view(torch.uint8) if t.dtype == E4M3 else t).copy_(u.view(torch.uint8) if u.dtype == E4M3 else u)
    torch.cuda.synchronize()
    for _ in range(3):
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
    torch.cuda.synchronize()
    for new, out in zip(other, outs):
        defs.check_product(out, *new)


@pytest.mark.parametrize("kind", KINDS)
def test_projection(kind):
    """QuantizedFp8 on rows, and on a residual's sum and norm; its codes and the result under them."""
    dtype, inputs, outputs, rows = KINDS[kind], 1000, 333, 37
    weight = torch.randn((outputs, inputs), generator=torch.Generator().manual_seed(1)).cuda() * inputs ** -0.5
    layer = ops.QuantizedFp8(weight)
    stored = layer.weight.float() * layer.scales.repeat_interleave(128, 0)[:outputs].repeat_interleave(128, 1)[:, :inputs]
    assert float((stored - weight).abs().max()) <= 2.0 ** -4 * float(weight.abs().max())
    x, residual = rows_of(rows, inputs, dtype, 7), rows_of(rows, inputs, dtype, 8)
    buffers = layer.buffers(rows)
    out = layer.forward(x, buffers=buffers)
    defs.check_product(out, *buffers, layer.weight, layer.scales)
    total = torch.empty_like(x)
    out = layer.forward_norm(x, None, residual=residual, sum_out=total, weight_offset=1.0, buffers=buffers)
    want, want_total = defs.norm_rows(x, residual, None, 1e-5, 1.0)
    assert torch.equal(total.cpu(), want_total)
    defs.check_codes(*buffers, want, NORM_ROUNDINGS)
    defs.check_product(out, *buffers, layer.weight, layer.scales)
    assert torch.equal(layer.forward(x), layer.forward(x, stream=torch.cuda.current_stream()))
    with pytest.raises(k.InvalidArgument):
        layer.forward(x[:, :999])


def test_projection_of_a_weight_that_is_trained():
    """A projection is a copy in codes: it keeps no graph of the weight that it was made from."""
    weight = torch.randn((40, 300), generator=torch.Generator().manual_seed(2)).cuda().requires_grad_()
    layer, plain = ops.QuantizedFp8(weight), ops.QuantizedFp8(weight.detach())
    assert not layer.scales.requires_grad and not layer.weight.requires_grad
    x = rows_of(5, 300, torch.bfloat16, 3)
    assert torch.equal(layer.forward(x), plain.forward(x))


def test_shape_and_type_refusals():
    t = torch.zeros((4, 128), dtype=torch.bfloat16, device="cuda")
    q, scale = torch.zeros((4, 128), dtype=E4M3, device="cuda"), torch.zeros((4, 1), device="cuda")
    for call in (lambda: ops.prepare_plain_fp8(t, q[:3], scale), lambda: ops.prepare_plain_fp8(t.float(), q, scale),
                 lambda: ops.prepare_plain_fp8(t, q, scale.double()), lambda: ops.prepare_plain_fp8(t.t(), q.t(), scale),
                 lambda: ops.prepare_norm_fp8(t, t, q, scale), lambda: ops.prepare_norm_fp8(t, None, q, scale, residual=t[:2]),
                 lambda: ops.prepare_norm_fp8(t, None, q, scale, sum_out=t), lambda: ops.gemm_fp8_128(q, scale, q, scale, t[:, :4]),
                 lambda: ops.gemm_fp8_128(q, scale, q, scale[:1], t), lambda: ops.gemm_fp8_128(q, scale, q, scale[:1], t[:, :4].float()),
                 lambda: ops.prepare_plain_fp8(t[:1].expand(4, 128), q, scale), lambda: ops.prepare_plain_fp8(t[:0], q[:0], scale[:0])):
        with pytest.raises(k.InvalidArgument):
            call()
