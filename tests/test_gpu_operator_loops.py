"""The e4m3, rotary and cross-attention operators at sizes where a block, a pair of CTAs or a warp walks several rows, tiles or
heads: the loops that a prompt or an image runs, which smaller sizes leave after one turn."""
import pytest
import torch

import operator_definitions as defs
from operator_definitions import KINDS

pytestmark = pytest.mark.gpu

k = pytest.importorskip("krea2_hrx_b200")
from krea2_hrx_b200 import ops  # noqa: E402

E4M3 = torch.float8_e4m3fn
NORM_ROUNDINGS = 60  # as in the tests of a few rows: the sums' order does not depend on how many there are


def multiprocessors():
    return torch.cuda.get_device_properties(0).multi_processor_count


def sample(rows, count):
    """The first rows, the last and some between."""
    return torch.unique(torch.cat([torch.arange(min(rows, count // 4)), torch.arange(max(0, rows - count // 4), rows),
                                   torch.linspace(0, rows - 1, count // 2).long()]))


def seeded(shape, dtype, seed, scale=1.0):
    """Made on the device: the values only have to differ from row to row."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(shape, generator=g, device="cuda") * scale).to(dtype)


def picked(t, rows):
    return t.view(torch.uint8)[rows].view(t.dtype) if t.dtype == E4M3 else t[rows]


# ------------------------------------------------------------------ codes
# Rows per SM that exceed the resident blocks several times (32 at most): three runs a thread, one warp, one run, single
# elements with one and two runs, two runs, the widest rows.
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("per_sm,width", [(13, 6144), (9, 4104), (70, 256), (50, 1000), (50, 1001), (20, 2056), (9, 8201), (9, 16384), (5, 32768)])
def test_a_block_walks_many_rows(kind, per_sm, width):
    dtype, rows = KINDS[kind], per_sm * multiprocessors() + 5
    x, residual = seeded((rows, width), dtype, 1), seeded((rows, width), dtype, 2, 3.0)
    x *= torch.linspace(0.25, 4.0, rows, device="cuda").to(dtype)[:, None]
    weights = seeded((width + 1,), torch.float32, 3, 0.1)
    rows_checked = sample(rows, max(16, 400000 // width))
    total = (x.float() + residual.float()).to(dtype)
    for weight in (None, weights[:width], weights[1:]):  # the last one off a 16-byte boundary
        for case in ("bare", "sum", "in place of x", "in place of the residual"):
            if weight is None and case != "bare":
                continue
            source, second = x.clone(), None if case == "bare" else residual.clone()
            target = {"bare": None, "sum": torch.empty_like(x), "in place of x": source, "in place of the residual": second}[case]
            q = torch.full((rows, -(-width // 16) * 16), 0x55, dtype=torch.uint8, device="cuda")
            scales = torch.full((rows, defs.groups(width)), -7.0, device="cuda")
            view = q.view(E4M3)[:, :width]
            ops.prepare_norm_fp8(source, weight, view, scales, residual=second, sum_out=target, weight_offset=1.0)
            at = rows_checked.cuda()
            want, _ = defs.norm_rows(x[at], None if second is None else residual[at], weight, 1e-5, 1.0)
            defs.check_codes(picked(view, at), scales[at], want, NORM_ROUNDINGS)
            assert bool((q[:, width:] == 0x55).all()) and bool((scales > 0).all())
            if target is not None:
                assert torch.equal(target, total)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("per_sm,width", [(9, 6144), (70, 256), (50, 1001), (9, 16384), (5, 32768)])
def test_a_block_walks_many_plain_rows(kind, per_sm, width):
    rows = per_sm * multiprocessors() + 5
    x = seeded((rows, width), KINDS[kind], 4)
    q = torch.empty((rows, -(-width // 16) * 16), dtype=E4M3, device="cuda")[:, :width]
    scales = torch.empty((rows, defs.groups(width)), device="cuda")
    ops.prepare_plain_fp8(x, q, scales)
    at = sample(rows, max(16, 400000 // width)).cuda()
    defs.check_codes(picked(q, at), scales[at], defs.f64(x[at]), 0)
    # the other rows against the same call on few rows, which a block leaves after one
    for first in range(0, rows, multiprocessors()):
        part = slice(first, min(rows, first + multiprocessors()))
        again = torch.empty((part.stop - first, q.stride(0)), dtype=E4M3, device="cuda")[:, :width], torch.empty_like(scales[part])
        ops.prepare_plain_fp8(x[part], *again)
        assert torch.equal(again[0].view(torch.uint8), q.view(torch.uint8)[part]) and torch.equal(again[1], scales[part])


# ------------------------------------------------------------------ product
def operands(m, n, width, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def codes(rows):
        buffer = torch.full((rows, -(-width // 16) * 16), 0x7f, dtype=torch.uint8, device="cuda")
        buffer[:, :width] = (torch.randn((rows, width), generator=g, device="cuda") * 60).clamp(-448, 448).to(E4M3).view(torch.uint8)
        return buffer.view(E4M3)[:, :width]

    def scales(rows):
        return torch.exp2(torch.rand((rows, defs.groups(width)), generator=g, device="cuda") * 6 - 12)

    return codes(m), scales(m), codes(n), scales(defs.groups(n))


# A pair's second and third tile with blocks that leave every phase of the rings; the last two in panels of columns (codes of
# a beyond 48 MB), the second one's last panel one tile wide.
@pytest.mark.parametrize("m,n,width,rows", [(2500, 5000, 300, 2500), (1300, 8001, 1100, 300), (2049, 6400, 129, 600), (3100, 3400, 16384, 48),
                                            (7001, 6915, 7200, 48)])
def test_a_pair_takes_many_tiles(m, n, width, rows):
    tiles = -(-m // 256) * -(-n // 256)
    assert tiles > multiprocessors() // 2 * 2
    a, a_scale, w, w_scale = operands(m, n, width, m)
    c = torch.full((m + 1, n + 3), 77.0, dtype=torch.bfloat16, device="cuda")
    ops.gemm_fp8_128(a, a_scale, w, w_scale, c[:m, :n])
    at = sample(m, rows).cuda()
    defs.check_product(c[at][:, :n], picked(a, at), a_scale[at], w, w_scale)
    assert bool((c[m] == 77.0).all()) and bool((c[:, n:] == 77.0).all())
    again = torch.full_like(c, 5.0)[:m, :n]
    ops.gemm_fp8_128(a, a_scale, w, w_scale, again)
    assert torch.equal(again.contiguous().view(torch.int16), c[:m, :n].contiguous().view(torch.int16))
    # the other rows: what leaves a tile's rows alone does not depend on the tiles in front of it
    part = slice(max(0, m - 1030), m)
    few = torch.empty((part.stop - part.start, n), dtype=torch.bfloat16, device="cuda")
    ops.gemm_fp8_128(picked(a, part), a_scale[part], w, w_scale, few)
    assert torch.equal(few.view(torch.int16), c[part, :n].contiguous().view(torch.int16)), "1030 rows take the same kernel"


# ------------------------------------------------------------------ rotary
# (dim, rotary_dim): pieces of 16 bytes; a part of the head; pairs (the partner not a whole number of pieces away); heads
# of more pieces than a warp has lanes; heads off 16-byte boundaries
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("layout", ["interleaved", "half"])
@pytest.mark.parametrize("tokens,q_heads,kv_heads,dim,rotary_dim", [(4609, 48, 12, 128, 128), (5000, 32, 8, 128, 96), (4801, 20, 3, 80, 80),
                                                                    (4801, 20, 3, 128, 34), (4737, 9, 2, 512, 512), (4737, 11, 5, 66, 34)])
def test_a_warp_walks_many_heads(kind, layout, tokens, q_heads, kv_heads, dim, rotary_dim):
    dtype = KINDS[kind]
    frequencies, magnitude = ops.rotary_frequencies(rotary_dim, scaling="parts", factor=4.0, trained=2048.0)
    positions = torch.arange(tokens, dtype=torch.int32, device="cuda") * 3 - 100
    q, kv = seeded((tokens, q_heads, dim), dtype, 1), seeded((tokens, kv_heads, dim), dtype, 2)
    at = sample(tokens, 32).cuda()
    for inverse in (False, True):
        def turn(*tensors, positions=positions):
            ops.rotary(*tensors, frequencies, positions=positions, magnitude=magnitude, layout=layout, inverse=inverse)

        q_out, k_out = torch.empty_like(q), torch.empty_like(kv)
        turn(q, kv, q_out, k_out)
        defs.check_rotary(q_out[at], q[at], positions[at].cpu(), frequencies, magnitude, layout, inverse)
        defs.check_rotary(k_out[at], kv[at], positions[at].cpu(), frequencies, magnitude, layout, inverse)
        in_place = q.clone(), kv.clone()
        turn(*in_place, *in_place)
        assert torch.equal(in_place[0], q_out) and torch.equal(in_place[1], k_out)
        # the other tokens against calls of few, whose warps take one head each
        for first in range(0, tokens, 500):
            part = slice(first, min(tokens, first + 60))
            few = torch.empty_like(q[part]), torch.empty_like(kv[part])
            turn(q[part], kv[part], *few, positions=positions[part])
            assert torch.equal(few[0], q_out[part]) and torch.equal(few[1], k_out[part])


# ------------------------------------------------------------------ cross attention
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("masked", [False, True])
def test_a_cta_walks_many_tiles_of_keys(kind, dim, masked):
    """Row tiles enough to fill the device, so that a CTA walks all 33 tiles of keys: the ring of mask words and the
    buffers of keys and values go round several times.  NaN and infinity lie in what does not count."""
    dtype, batch, q_len, kv_len, heads = KINDS[kind], 3, 1043, 4109, 16
    q, key, value = seeded((batch, q_len, heads, dim), dtype, 1), seeded((batch, kv_len, heads, dim), dtype, 2), seeded((batch, kv_len, heads, dim), dtype, 3)
    lengths = torch.tensor([kv_len, 0, 2900], dtype=torch.int32)
    counts = torch.arange(kv_len) < lengths[:, None]
    mask = None
    if masked:
        mask = torch.rand((batch, kv_len), generator=torch.Generator().manual_seed(4)) < 0.8
        mask[0, 128:640] = False  # whole tiles in which no key counts, in front of others, between them and at the end
        mask[2, :300] = False
        mask[0, 4000:] = False
        counts &= mask
    key[~counts.cuda()], value[~counts.cuda()] = float("nan"), float("inf")
    out = torch.full_like(q, 9.0)
    ops.cross_attention(q, key, value, out, kv_lengths=lengths.cuda(), key_mask=None if mask is None else mask.cuda())
    at = sample(q_len, 40).cuda()
    defs.check_cross(out[:, at], q[:, at], key, value, dim ** -0.5, lengths, mask)
    assert bool(torch.isfinite(out).all()) and not bool(out[1].float().any())
    # the other queries against calls of one row tile, whose keys are split over several CTAs: the same up to the roundings
    # of either (bf16 2^-8, f16 2^-11 of the weights and of the result, each way) of values of at most 6
    step = 4 * defs.HALF_STEP[dtype] * 6.0
    for first in range(0, q_len, 128):
        part = slice(first, min(q_len, first + 128))
        few = torch.empty_like(q[:, part])
        ops.cross_attention(q[:, part], key, value, few, kv_lengths=lengths.cuda(), key_mask=None if mask is None else mask.cuda())
        assert float((few.float() - out[:, part].float()).abs().max()) <= step
    assert k.device_status() == 0
