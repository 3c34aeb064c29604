"""What the e4m3 projection, rotary and cross-attention entry points refuse, and the rotary frequencies: host work, no
device is touched."""
import ctypes

import pytest
import torch

import krea2_hrx_b200 as k
import operator_definitions as defs
from krea2_hrx_b200 import ops

NORM = dict(stream=None, tokens=3, x="p", residual=None, weight=None, sum=None, q="p", q_scale="p", width=256, x_stride=256, residual_stride=0,
            sum_stride=0, out_stride=256, eps=1e-5, weight_offset=0.0, kind=1)
PLAIN = dict(stream=None, tokens=3, x="p", q="p", q_scale="p", width=256, x_stride=256, out_stride=256, kind=1)
GEMM = dict(stream=None, m=3, a="p", w="p", scale="p", a_scale="p", c="p", k_size=256, a_stride=256, w_stride=256, n_size=40, c_stride=40, kind=0)
ROTARY = dict(stream=None, tokens=3, q="p", k="p", positions=None, frequencies="p", q_out="p", k_out="p", q_heads=4, kv_heads=2, head_dim=64,
              rotary_dim=64, q_stride=256, k_stride=128, q_out_stride=256, k_out_stride=128, magnitude=1.0, layout=0, inverse=0, kind=0)
CROSS = dict(stream=None, batch=2, q_len=5, kv_len=7, q="p", k="p", v="p", kv_lengths=None, key_mask=None, out="p", q_heads=4, kv_heads=2,
             head_dim=64, q_batch_stride=1280, q_stride=256, k_batch_stride=896, k_stride=128, v_batch_stride=896, v_stride=128,
             out_batch_stride=1280, out_stride=256, mask_stride=0, scale=0.125, kind=1)
CALLS = {"krea2_prepare_norm_fp8": NORM, "krea2_prepare_plain_fp8": PLAIN, "krea2_gemm_fp8_128": GEMM, "krea2_rotary": ROTARY,
         "krea2_cross_attention": CROSS}

REFUSED = [
    ("krea2_prepare_norm_fp8", dict(tokens=0), "tokens"), ("krea2_prepare_norm_fp8", dict(width=0), "width"),
    ("krea2_prepare_norm_fp8", dict(width=32769, x_stride=40000, out_stride=40000), "width"),
    ("krea2_prepare_norm_fp8", dict(x_stride=255), "x_stride"), ("krea2_prepare_norm_fp8", dict(out_stride=264), "out_stride"),
    ("krea2_prepare_norm_fp8", dict(out_stride=240), "out_stride"), ("krea2_prepare_norm_fp8", dict(kind=2), "kind"),
    ("krea2_prepare_norm_fp8", dict(x=None), "null"), ("krea2_prepare_norm_fp8", dict(q="p+8"), "aligned"),
    ("krea2_prepare_norm_fp8", dict(x="p+1"), "aligned"), ("krea2_prepare_norm_fp8", dict(eps=-1.0), "eps"),
    ("krea2_prepare_norm_fp8", dict(eps=float("nan")), "eps"), ("krea2_prepare_norm_fp8", dict(weight_offset=float("inf")), "weight_offset"),
    ("krea2_prepare_norm_fp8", dict(sum="p", sum_stride=256), "residual"), ("krea2_prepare_norm_fp8", dict(residual="p", residual_stride=8), "residual_stride"),
    ("krea2_prepare_norm_fp8", dict(residual="p", residual_stride=256, sum="p", sum_stride=8), "sum_stride"),
    ("krea2_prepare_plain_fp8", dict(tokens=1 << 25), "tokens"), ("krea2_prepare_plain_fp8", dict(q_scale="p+2"), "aligned"),
    ("krea2_prepare_plain_fp8", dict(kind=-1), "kind"), ("krea2_prepare_plain_fp8", dict(q=None), "null"),
    ("krea2_gemm_fp8_128", dict(m=0), "m 0"), ("krea2_gemm_fp8_128", dict(k_size=0), "k_size"), ("krea2_gemm_fp8_128", dict(n_size=0), "n_size"),
    ("krea2_gemm_fp8_128", dict(n_size=262145, c_stride=262145), "n_size"), ("krea2_gemm_fp8_128", dict(k_size=65537, a_stride=65552, w_stride=65552), "k_size"),
    ("krea2_gemm_fp8_128", dict(a_stride=264), "a_stride"), ("krea2_gemm_fp8_128", dict(w_stride=240), "w_stride"),
    ("krea2_gemm_fp8_128", dict(c_stride=39), "c_stride"), ("krea2_gemm_fp8_128", dict(kind=2), "kind"), ("krea2_gemm_fp8_128", dict(w="p+4"), "aligned"),
    ("krea2_gemm_fp8_128", dict(c="p+1"), "aligned"), ("krea2_gemm_fp8_128", dict(a_scale=None), "null"),
    ("krea2_rotary", dict(tokens=0), "tokens"), ("krea2_rotary", dict(q_heads=0), "heads"), ("krea2_rotary", dict(rotary_dim=66), "rotary_dim"),
    ("krea2_rotary", dict(rotary_dim=63), "rotary_dim"), ("krea2_rotary", dict(rotary_dim=0), "rotary_dim"),
    ("krea2_rotary", dict(head_dim=514, rotary_dim=64), "head_dim"), ("krea2_rotary", dict(q_stride=255), "strides"),
    ("krea2_rotary", dict(k_out_stride=127), "strides"), ("krea2_rotary", dict(magnitude=float("nan")), "magnitude"),
    ("krea2_rotary", dict(layout=2), "layout"), ("krea2_rotary", dict(inverse=2), "inverse"), ("krea2_rotary", dict(kind=3), "kind"),
    ("krea2_rotary", dict(k=None), "null"), ("krea2_rotary", dict(frequencies=None), "null"), ("krea2_rotary", dict(frequencies="p+4"), "aligned"),
    ("krea2_rotary", dict(q_out_stride=512), "in place"), ("krea2_rotary", dict(k_out_stride=512), "in place"),
    ("krea2_cross_attention", dict(batch=0), "batch"), ("krea2_cross_attention", dict(batch=65536), "batch"), ("krea2_cross_attention", dict(q_len=0), "q_len"),
    ("krea2_cross_attention", dict(kv_len=1 << 25), "kv_len"), ("krea2_cross_attention", dict(kv_heads=3), "heads"),
    ("krea2_cross_attention", dict(kv_heads=0), "heads"), ("krea2_cross_attention", dict(head_dim=136), "head_dim"),
    ("krea2_cross_attention", dict(head_dim=60), "head_dim"), ("krea2_cross_attention", dict(q_stride=248), "strides"),
    ("krea2_cross_attention", dict(k_stride=120), "strides"), ("krea2_cross_attention", dict(v_stride=132), "multiples of 8"),
    ("krea2_cross_attention", dict(k_batch_stride=900), "multiples of 8"), ("krea2_cross_attention", dict(out_batch_stride=256), "overlap"),
    ("krea2_prepare_norm_fp8", dict(residual="p+16", residual_stride=256, sum="p", sum_stride=512), "in place"),
    ("krea2_prepare_norm_fp8", dict(residual="p+16", residual_stride=256, sum="p+16", sum_stride=512), "in place"),
    ("krea2_cross_attention", dict(q_heads=258, head_dim=8, q_stride=2064, out_stride=2064, q_batch_stride=16384, out_batch_stride=16384), "share a key head"),
    ("krea2_cross_attention", dict(out_batch_stride=0), "overlap"), ("krea2_cross_attention", dict(out_batch_stride=248, out_stride=512), "overlap"),
    ("krea2_cross_attention", dict(key_mask="p", mask_stride=6), "mask_stride"), ("krea2_cross_attention", dict(scale=0.0), "scale"),
    ("krea2_cross_attention", dict(scale=float("nan")), "scale"), ("krea2_cross_attention", dict(scale=-1.0), "scale"),
    ("krea2_cross_attention", dict(kind=2), "kind"), ("krea2_cross_attention", dict(v=None), "null"), ("krea2_cross_attention", dict(q="p+8"), "aligned"),
    ("krea2_cross_attention", dict(kv_lengths="p+2"), "aligned"),
]


@pytest.mark.parametrize("name,change,needle", REFUSED)
def test_bad_arguments_are_refused_before_any_device_work(name, change, needle):
    buffer = ctypes.create_string_buffer(64)
    base = (ctypes.addressof(buffer) + 15) & ~15
    args = [base + int(value[2:] or 0) if isinstance(value, str) else value for value in {**CALLS[name], **change}.values()]
    assert getattr(k.lib(), name)(*args) == 1
    message = k.lib().krea2_last_error().decode()
    assert needle in message and message.startswith(name[len("krea2_"):]), message


@pytest.mark.parametrize("call", [
    lambda t, f: ops.prepare_plain_fp8(t(4, 128), t(4, 128, d=torch.float8_e4m3fn), t(4, 1, d=torch.float32)),
    lambda t, f: ops.prepare_norm_fp8(t(4, 128, d=torch.float32), None, t(4, 128), t(4, 1)),
    lambda t, f: ops.gemm_fp8_128(t(4, 128, d=torch.float8_e4m3fn), t(4, 1, d=torch.float32), t(8, 128, d=torch.float8_e4m3fn),
                                  t(1, 1, d=torch.float32), t(4, 8)),
    lambda t, f: ops.rotary(t(3, 2, 64), None, t(3, 2, 64), None, f),
    lambda t, f: ops.cross_attention(t(1, 2, 2, 64), t(1, 3, 2, 64), t(1, 3, 2, 64), t(1, 2, 2, 64)),
    lambda t, f: ops.QuantizedFp8(t(4, 128)),
])
def test_host_tensors_are_refused(call):
    with pytest.raises(k.InvalidArgument):
        call(lambda *shape, d=torch.bfloat16: torch.zeros(shape).to(d), torch.zeros(32, dtype=torch.float64))


@pytest.mark.parametrize("rotary_dim", [2, 6, 64, 128])
@pytest.mark.parametrize("scaling", ["none", "linear", "base", "parts"])
def test_rotary_frequencies(rotary_dim, scaling):
    got, magnitude = ops.rotary_frequencies(rotary_dim, 10000.0, scaling, factor=8.0, trained=4096.0, device="cpu")
    want, want_magnitude = defs.frequencies_of(rotary_dim, 10000.0, scaling, 8.0, 4096.0, 1.0, 32.0)
    # pow and the few products around it: some roundings of 2^-53
    assert torch.allclose(got, torch.tensor(want, dtype=torch.float64), rtol=64 * 2.0 ** -53, atol=0.0)
    assert abs(magnitude - want_magnitude) <= defs.F32 * want_magnitude
    if scaling == "base" and rotary_dim > 2:
        plain, _ = ops.rotary_frequencies(rotary_dim, 10000.0, device="cpu")
        assert got[0] == 1.0 and abs(float(got[-1] / plain[-1]) - 1 / 8) < 1e-12  # the slowest is divided by the factor


def test_rotary_frequencies_refusals():
    for bad in (dict(rotary_dim=3), dict(rotary_dim=0), dict(rotary_dim=514), dict(base=1.0), dict(base=float("inf")), dict(scaling="other"),
                dict(scaling="linear", factor=0.5), dict(scaling="parts", factor=2.0, trained=0.0),
                dict(scaling="parts", factor=2.0, trained=100.0, slow=4.0, fast=4.0), dict(scaling="base", factor=1e300)):
        with pytest.raises(k.InvalidArgument):
            ops.rotary_frequencies(**{"rotary_dim": 64, "device": "cpu", **bad})
