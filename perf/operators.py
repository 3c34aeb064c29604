"""Cases of the e4m3 projection path, the rotary positions and the cross attention: inputs, plain forms and the library's calls.

A cross-attention sublayer beside the W8A8 block: the residual's addition and the RMS norm write e4m3 codes with one scale
per 128 channels, the e4m3 product reads them against weights with one scale per 128 x 128 block, the rotary positions turn
queries and keys, and the queries attend to an encoder's states of another length.  Each case names its operator in "op":

  norm    sum = T(x + residual), codes and scales of sum / rms(sum) * (offset + weight)
  plain   codes and scales of the rows as they are
  gemm    c = T(sum over k blocks of a_scale * w_scale * (codes . codes))
  rotary  queries and keys turned by position * frequency, forwards or (inverse) backwards
  cross   softmax(scale q . k over the keys that count) v, zero where no key counts

Sizes follow the session's dimensions (width 6144, 48 / 12 heads of 128, SwiGLU width 16384, 4096 or 16384 image tokens
beside 512 text tokens) and the kernel bench's row counts (1043, 4109).
"""
import math

import torch

own = False

E4M3_MAX = 448.0
BLOCK = 128
TYPES = {"bf16": torch.bfloat16, "f16": torch.float16}
LARGEST_PRODUCT = 4608 * 15360 * 6144
LARGEST_SCORES = 48 * 16384 * 512


def listed():
    return [
        # one token of a text model's decoding step: latency
        {"name": "norm token", "op": "norm", "rows": 1, "width": 6144, "type": "bf16", "residual": True},
        # a 1024 x 1024 image with its text tokens
        {"name": "norm image", "op": "norm", "rows": 4608, "width": 6144, "type": "bf16", "residual": True},
        # the down projection's input at a ragged row count of the kernel bench
        {"name": "plain ragged", "op": "plain", "rows": 1043, "width": 16384, "type": "f16"},
        # one token through a square projection: the weights' bytes are all there is
        {"name": "gemm token", "op": "gemm", "m": 1, "n": 6144, "k": 6144, "type": "bf16"},
        # the encoder's ragged batch through the down projection
        {"name": "gemm ragged", "op": "gemm", "m": 275, "n": 6144, "k": 16384, "type": "f16"},
        # q|k|v|gate of a 1024 x 1024 image
        {"name": "gemm image", "op": "gemm", "m": 4608, "n": 15360, "k": 6144, "type": "bf16"},
        # one token, queries and keys
        {"name": "rotary token", "op": "rotary", "tokens": 1, "q_heads": 48, "kv_heads": 12, "head_dim": 128, "rotary_dim": 128,
         "layout": "interleaved", "inverse": False, "scaling": "none", "first": 4608, "type": "f16"},
        # the image's queries and keys
        {"name": "rotary image", "op": "rotary", "tokens": 4608, "q_heads": 48, "kv_heads": 12, "head_dim": 128, "rotary_dim": 128,
         "layout": "interleaved", "inverse": False, "scaling": "none", "first": 0, "type": "f16"},
        # a long text far into its context, half layout on a part of the head, turned back
        {"name": "rotary far inverse", "op": "rotary", "tokens": 12301, "q_heads": 32, "kv_heads": 8, "head_dim": 128, "rotary_dim": 96,
         "layout": "half", "inverse": True, "scaling": "parts", "first": 1000003, "type": "bf16"},
        # one query each of a small batch against a prompt's states
        {"name": "cross token", "op": "cross", "batch": 2, "q_len": 1, "kv_len": 512, "q_heads": 48, "kv_heads": 12, "head_dim": 128,
         "lengths": True, "mask": False, "type": "bf16"},
        # a padded batch with a tokenizer's mask, one of whose prompts is empty
        {"name": "cross ragged", "op": "cross", "batch": 3, "q_len": 1043, "kv_len": 4109, "q_heads": 16, "kv_heads": 16, "head_dim": 64,
         "lengths": True, "mask": True, "type": "f16"},
        # a 2048 x 2048 image against its prompt
        {"name": "cross image", "op": "cross", "batch": 1, "q_len": 16384, "kv_len": 512, "q_heads": 48, "kv_heads": 12, "head_dim": 128,
         "lengths": False, "mask": False, "type": "bf16"},
    ]


def _log(rng, low, high):
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high + 1)))))))


def draw(rng):
    op = rng.choice(["norm", "plain", "gemm", "gemm", "rotary", "rotary", "cross", "cross"])
    kind = rng.choice(["bf16", "f16"])
    if op in ("norm", "plain"):
        width = _log(rng, 64, 16384)
        rows = _log(rng, 1, min(16896, 4608 * 6144 // width))
        case = {"op": op, "rows": rows, "width": width, "type": kind}
        return dict(case, residual=rng.random() < 0.75) if op == "norm" else case
    if op == "gemm":
        m, k = _log(rng, 1, 8192), _log(rng, 64, 16384)
        return {"op": op, "m": m, "n": _log(rng, 64, min(32768, LARGEST_PRODUCT // (m * k))), "k": k, "type": kind}
    if op == "rotary":
        head_dim = rng.choice([64, 80, 96, 128, 256])
        kv_heads = rng.choice([1, 2, 8, 12])
        q_heads = kv_heads * rng.choice([1, 2, 4])
        rotary_dim = rng.choice([head_dim, head_dim // 2, 2 * rng.randint(1, head_dim // 2)])
        most = 12301 * 40 * 128 // ((q_heads + kv_heads) * head_dim)
        return {"op": op, "tokens": _log(rng, 1, min(16896, most)), "q_heads": q_heads, "kv_heads": kv_heads, "head_dim": head_dim,
                "rotary_dim": rotary_dim, "layout": rng.choice(["interleaved", "half"]), "inverse": rng.random() < 0.5,
                "scaling": rng.choice(["none", "linear", "base", "parts"]), "first": rng.choice([0, _log(rng, 1, 4000000)]), "type": kind}
    batch, kv_heads = _log(rng, 1, 8), rng.choice([1, 4, 8, 12, 16])
    q_heads = kv_heads * rng.choice([1, 2, 3, 4])
    kv_len = _log(rng, 1, 8192)
    most = max(1, LARGEST_SCORES // (batch * q_heads * kv_len))
    q_len = rng.choice([1, _log(rng, 1, min(16384, most))])
    return {"op": op, "batch": batch, "q_len": q_len, "kv_len": kv_len, "q_heads": q_heads, "kv_heads": kv_heads,
            "head_dim": rng.choice([40, 64, 80, 128]), "lengths": rng.random() < 0.6, "mask": rng.random() < 0.4, "type": kind}


# ------------------------------------------------------------------ inputs
def _activations(rows, width, dtype, generator):
    """~N(0, 1) with one channel in a hundred twenty times larger."""
    x = torch.randn((rows, width), generator=generator, device="cuda")
    large = torch.rand(width, generator=generator, device="cuda") < 0.01
    return (x * torch.where(large, 20.0, 1.0)).to(dtype)


def _groups(width):
    return -(-width // BLOCK)


def _codes_of(x):
    """e4m3 codes of f32 rows and their scales, one per 128 channels."""
    rows, width = x.shape
    padded = torch.nn.functional.pad(x, (0, _groups(width) * BLOCK - width)).view(rows, -1, BLOCK)
    scale = (padded.abs().amax(-1) / E4M3_MAX).clamp_min(2.0 ** -126)
    codes = (padded * (1.0 / scale)[..., None]).clamp(-E4M3_MAX, E4M3_MAX).reshape(rows, -1)[:, :width]
    return codes.to(torch.float8_e4m3fn), scale


def _pitched(codes):
    """The same codes in rows whose pitch is a multiple of 16 bytes."""
    rows, width = codes.shape
    buffer = torch.zeros((rows, -(-width // 16) * 16), dtype=torch.uint8, device=codes.device)
    buffer[:, :width] = codes.view(torch.uint8)
    return buffer.view(torch.float8_e4m3fn)[:, :width]


def _frequencies(case):
    """Radians per position of each pair, in f64: 1 / base^(2 i / rotary_dim), scaled for a context eight times 4096."""
    half, base, factor, trained = case["rotary_dim"] // 2, 10000.0, 8.0, 4096.0
    if case["scaling"] == "base":
        base *= factor ** (case["rotary_dim"] / max(1, case["rotary_dim"] - 2))
    i = torch.arange(half, dtype=torch.float64)
    plain = base ** (-2.0 * i / case["rotary_dim"])
    if case["scaling"] == "linear":
        return plain / factor, 1.0
    if case["scaling"] == "parts":
        turns = trained * plain / (2.0 * math.pi)
        kept = ((turns - 1.0) / (32.0 - 1.0)).clamp(0.0, 1.0)
        return plain * kept + plain / factor * (1.0 - kept), 0.1 * math.log(factor) + 1.0
    return plain, 1.0


def prepare(case, seed):
    generator = torch.Generator(device="cuda").manual_seed(seed)
    dtype = TYPES[case["type"]]
    state = {"case": case}
    if case["op"] in ("norm", "plain"):
        rows, width = case["rows"], case["width"]
        state["x"] = _activations(rows, width, dtype, generator)
        if case["op"] == "norm":
            state["residual"] = _activations(rows, width, dtype, generator) if case["residual"] else None
            state["weight"] = torch.randn(width, generator=generator, device="cuda") * 0.1
            state["sum"] = torch.empty_like(state["x"]) if case["residual"] else None
        state["q"] = torch.empty((rows, -(-width // 16) * 16), dtype=torch.float8_e4m3fn, device="cuda")[:, :width]
        state["q_scale"] = torch.empty((rows, _groups(width)), dtype=torch.float32, device="cuda")
    elif case["op"] == "gemm":
        m, n, k = case["m"], case["n"], case["k"]
        codes, state["a_scale"] = _codes_of(_activations(m, k, torch.float32, generator))
        state["a"] = _pitched(codes)
        w = torch.randn((n, k), generator=generator, device="cuda").mul_(k ** -0.5)
        blocks = torch.nn.functional.pad(w, (0, _groups(k) * BLOCK - k, 0, _groups(n) * BLOCK - n)).view(_groups(n), BLOCK, _groups(k), BLOCK)
        state["w_scale"] = (blocks.abs().amax((1, 3)) / E4M3_MAX).clamp_min(2.0 ** -126)
        scaled = (blocks / state["w_scale"][:, None, :, None]).clamp(-E4M3_MAX, E4M3_MAX)
        state["w"] = _pitched(scaled.reshape(_groups(n) * BLOCK, -1)[:n, :k].to(torch.float8_e4m3fn))
        state["c"] = torch.empty((m, n), dtype=dtype, device="cuda")
    elif case["op"] == "rotary":
        tokens, head_dim = case["tokens"], case["head_dim"]
        state["q"] = torch.randn((tokens, case["q_heads"], head_dim), generator=generator, device="cuda").to(dtype)
        state["k"] = torch.randn((tokens, case["kv_heads"], head_dim), generator=generator, device="cuda").to(dtype)
        state["positions"] = torch.arange(case["first"], case["first"] + tokens, dtype=torch.int32, device="cuda")
        frequencies, state["magnitude"] = _frequencies(case)
        state["frequencies"] = frequencies.cuda()
        state["q_out"], state["k_out"] = torch.empty_like(state["q"]), torch.empty_like(state["k"])
    else:
        batch, q_len, kv_len, d = case["batch"], case["q_len"], case["kv_len"], case["head_dim"]
        state["q"] = torch.randn((batch, q_len, case["q_heads"], d), generator=generator, device="cuda").to(dtype)
        state["k"] = torch.randn((batch, kv_len, case["kv_heads"], d), generator=generator, device="cuda").to(dtype)
        state["v"] = torch.randn((batch, kv_len, case["kv_heads"], d), generator=generator, device="cuda").to(dtype)
        state["lengths"] = state["mask"] = None
        if case["lengths"]:
            state["lengths"] = torch.randint(0, kv_len + 1, (batch,), generator=generator, device="cuda", dtype=torch.int32)
            state["lengths"][0] = kv_len
            if batch > 2:
                state["lengths"][1] = 0
        if case["mask"]:
            state["mask"] = torch.rand((batch, kv_len), generator=generator, device="cuda") < 0.8
        state["scale"] = d ** -0.5
        state["out"] = torch.empty_like(state["q"])
    return state


# ------------------------------------------------------------------ one pass
def run(state):
    return _calls(state) if own else _plain(state)


def _calls(state):
    from krea2_hrx_b200 import ops
    op = state["case"]["op"]
    if op == "norm":
        ops.prepare_norm_fp8(state["x"], state["weight"], state["q"], state["q_scale"], residual=state["residual"], sum_out=state["sum"],
                             eps=1e-5, weight_offset=1.0)
        out = {"q": state["q"], "q_scale": state["q_scale"]}
        return dict(out, sum=state["sum"]) if state["residual"] is not None else out
    if op == "plain":
        ops.prepare_plain_fp8(state["x"], state["q"], state["q_scale"])
        return {"q": state["q"], "q_scale": state["q_scale"]}
    if op == "gemm":
        ops.gemm_fp8_128(state["a"], state["a_scale"], state["w"], state["w_scale"], state["c"])
        return state["c"]
    if op == "rotary":
        ops.rotary(state["q"], state["k"], state["q_out"], state["k_out"], state["frequencies"], positions=state["positions"],
                   magnitude=state["magnitude"], layout=state["case"]["layout"], inverse=state["case"]["inverse"])
        return {"q": state["q_out"], "k": state["k_out"]}
    ops.cross_attention(state["q"], state["k"], state["v"], state["out"], kv_lengths=state["lengths"], key_mask=state["mask"],
                        scale=state["scale"])
    return state["out"]


def _turned(x, cos, sin, case):
    """x [tokens][heads][head_dim] in f32 or f64, cos and sin [tokens][1][rotary_dim / 2] of the same type."""
    r = case["rotary_dim"]
    if case["layout"] == "interleaved":
        a, b = x[..., 0:r:2], x[..., 1:r:2]
        turned = torch.stack((a * cos - b * sin, b * cos + a * sin), dim=-1).flatten(-2)
    else:
        a, b = x[..., : r // 2], x[..., r // 2: r]
        turned = torch.cat((a * cos - b * sin, b * cos + a * sin), dim=-1)
    return torch.cat((turned, x[..., r:]), dim=-1)


def _counting(state):
    """[batch][1][1][1][kv_len], true where a key counts; None where all do."""
    case, counts = state["case"], None
    if state["lengths"] is not None:
        counts = torch.arange(case["kv_len"], device="cuda") < state["lengths"][:, None]
    if state["mask"] is not None:
        counts = state["mask"] if counts is None else counts & state["mask"]
    return None if counts is None else counts[:, None, None, None, :]


def _attended(q, k, v, counts, scale, case):
    """All in the type of q: [batch][q_len][q_heads][d]."""
    batch, q_len, kv_heads = case["batch"], case["q_len"], case["kv_heads"]
    shares = case["q_heads"] // kv_heads
    q = q.view(batch, q_len, kv_heads, shares, -1).permute(0, 2, 3, 1, 4)
    k, v = (t.permute(0, 2, 1, 3)[:, :, None] for t in (k, v))
    scores = torch.matmul(q, k.transpose(-1, -2)).mul_(scale)
    if counts is not None:
        scores = scores.masked_fill(~counts, -math.inf)
    top = scores.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, torch.zeros_like(top), top)
    weights = scores.sub_(top).exp_()
    total = weights.sum(-1, keepdim=True)
    out = torch.matmul(weights, v) / torch.where(total == 0, torch.ones_like(total), total)
    return out.permute(0, 3, 1, 2, 4).reshape(batch, q_len, case["q_heads"], -1)


def _plain(state):
    case = state["case"]
    dtype = TYPES[case["type"]]
    if case["op"] in ("norm", "plain"):
        x = state["x"].float()
        if case["op"] == "plain":
            q, scale = _codes_of(x)
            return {"q": q, "q_scale": scale}
        if state["residual"] is not None:
            total = (x + state["residual"].float()).to(dtype)
            x = total.float()
        y = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-5) * (1.0 + state["weight"])
        q, scale = _codes_of(y)
        out = {"q": q, "q_scale": scale}
        return dict(out, sum=total) if state["residual"] is not None else out
    if case["op"] == "gemm":
        a = state["a"].float() * state["a_scale"].repeat_interleave(BLOCK, 1)[:, : case["k"]]
        w = state["w"].float() * state["w_scale"].repeat_interleave(BLOCK, 0)[: case["n"]].repeat_interleave(BLOCK, 1)[:, : case["k"]]
        return torch.matmul(a, w.t()).to(dtype)
    if case["op"] == "rotary":
        angles = state["positions"].double()[:, None] * state["frequencies"]
        cos, sin = (angles.cos() * state["magnitude"]).float()[:, None], (angles.sin() * state["magnitude"]).float()[:, None]
        if case["inverse"]:
            sin = -sin
        return {name: _turned(state[name].float(), cos, sin, case).to(dtype) for name in ("q", "k")}
    return _attended(state["q"].float(), state["k"].float(), state["v"].float(), _counting(state), state["scale"], case).to(dtype)


# ------------------------------------------------------------------ what a pass has to do
def work(case):
    if case["op"] in ("norm", "plain"):
        values = case["rows"] * case["width"]
        read = values * (4 if case.get("residual") else 2) + (case["width"] * 4 if case["op"] == "norm" else 0)
        written = values * (3 if case.get("residual") else 1) + case["rows"] * _groups(case["width"]) * 4
        return {"bytes": read + written, "flops": values * (8 if case["op"] == "norm" else 3)}
    if case["op"] == "gemm":
        m, n, k = case["m"], case["n"], case["k"]
        scales = 4 * _groups(k) * (m + _groups(n))
        return {"bytes": m * k + n * k + 2 * m * n + scales, "flops": 2 * m * n * k}
    if case["op"] == "rotary":
        values = case["tokens"] * (case["q_heads"] + case["kv_heads"]) * case["head_dim"]
        turned = values // case["head_dim"] * case["rotary_dim"]
        return {"bytes": 4 * values + 4 * case["tokens"] + 4 * case["rotary_dim"], "flops": 3 * turned}
    b, q, kv = case["batch"], case["q_len"], case["kv_len"]
    # the first length is kv_len, the second of three or more is 0, the others are any of 0 .. kv_len
    share = (1.0 + max(0, b - (2 if b > 2 else 1)) / 2) / b if case["lengths"] else 1.0
    moved = 2 * b * q * case["q_heads"] * case["head_dim"] * 2 + share * 2 * b * kv * case["kv_heads"] * case["head_dim"] * 2
    return {"bytes": moved + (b * kv if case["mask"] else 0), "flops": share * 4 * b * q * kv * case["q_heads"] * case["head_dim"]}


# ------------------------------------------------------------------ the definition in 64 bits
def exact(case, seed):
    state = prepare(case, seed)
    op = case["op"]
    if op in ("norm", "plain"):
        rows, width = case["rows"], case["width"]
        y, out = state["x"].double(), {}
        if op == "norm":
            if state["residual"] is not None:
                out["sum"] = y + state["residual"].double()
                y = out["sum"].to(TYPES[case["type"]]).double()  # the norm is taken of the rounded sum
            y = y / (y.pow(2).sum(-1, keepdim=True) / width + 1e-5).sqrt() * (state["weight"].double() + 1.0)
        out["q"], out["q_scale"] = torch.empty_like(y), torch.empty((rows, _groups(width)), dtype=torch.float64, device="cuda")
        for g in range(_groups(width)):
            part = y[:, g * BLOCK: (g + 1) * BLOCK]
            out["q_scale"][:, g] = (part.abs().max(-1).values / E4M3_MAX).clamp_min(2.0 ** -126)
            out["q"][:, g * BLOCK: (g + 1) * BLOCK] = part / out["q_scale"][:, g: g + 1]
        return out
    if op == "gemm":
        c = torch.zeros((case["m"], case["n"]), dtype=torch.float64, device="cuda")
        wide = torch.arange(case["n"], device="cuda") // BLOCK
        for g in range(_groups(case["k"])):
            at = slice(g * BLOCK, (g + 1) * BLOCK)
            w = state["w"][:, at].to(torch.float64) * state["w_scale"].double()[wide, g][:, None]
            c.addmm_(state["a"][:, at].to(torch.float64) * state["a_scale"][:, g: g + 1].double(), w.t())
        return c
    if op == "rotary":
        angle = torch.outer(state["positions"].double(), state["frequencies"])
        turn = torch.polar(torch.full_like(angle, state["magnitude"]), -angle if case["inverse"] else angle)[:, None, :]
        half, out = case["rotary_dim"] // 2, {}
        for name in ("q", "k"):
            x = state[name].double()
            first, second = (slice(0, 2 * half, 2), slice(1, 2 * half, 2)) if case["layout"] == "interleaved" else (slice(0, half), slice(half, 2 * half))
            z = torch.complex(x[..., first], x[..., second]) * turn
            x[..., first], x[..., second] = z.real, z.imag
            out[name] = x
        return out
    shares, out = case["q_heads"] // case["kv_heads"], torch.zeros(state["q"].shape, dtype=torch.float64, device="cuda")
    for b in range(case["batch"]):
        kept = torch.ones(case["kv_len"], dtype=torch.bool, device="cuda")
        if state["lengths"] is not None:
            kept[int(state["lengths"][b]):] = False
        if state["mask"] is not None:
            kept &= state["mask"][b]
        if not bool(kept.any()):
            continue
        for h in range(case["q_heads"]):
            k, v = (state[name][b, kept, h // shares].double() for name in ("k", "v"))
            out[b, :, h] = torch.softmax(state["q"][b, :, h].double() @ k.t() * state["scale"], -1) @ v
    return out
