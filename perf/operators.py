"""What is measured of the operators around a parallel layer's folds and copies, and how.

Two pairs of operators.  The norms around a block, fused with the fold of its partial outputs, its gate and its
residual scale, and their backward pass:

    y = sum_k in_k          n = post(y)          r = residual_scale * x + block_scale * gate * n          h = pre(r)

and a cache of keys and values held in blocks of 32 elements with a shared power-of-two scale (8 or 4 bits an
element), written token by token and read back through page tables.

`own = False` computes them in elementary torch operations, `own = True` through ``pccl_amd.hip``.
"""
import math

import torch

own = False

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
BYTES = {"f32": 4, "bf16": 2, "f16": 2}

# A cache format's elements: smallest binary exponent of a step's binade, mantissa bits, largest value and its exponent.
# i8 holds k / 64, |k| <= 127: one binade of seven fractional bits' grid, written here as exponent 0 with 6 mantissa bits.
FORMATS = {"f8e4m3": dict(emin=-6, mbits=3, top=448.0, emax=8, bits=8),
           "f8e5m2": dict(emin=-14, mbits=2, top=57344.0, emax=15, bits=8),
           "i8": dict(emin=0, mbits=6, top=127 / 64, emax=0, bits=8),
           "f4e2m1": dict(emin=0, mbits=1, top=6.0, emax=2, bits=4)}
F4_VALUES = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0, -0.0, -0.5, -1.0, -1.5, -2.0, -3.0, -4.0, -6.0)
BLOCK = 32


# ---- the cases -----------------------------------------------------------------------------------------------------

def _norm(op, name, dtype, rows, width, n_in, n_out, post, pre, gate_rows, bias, params, offset, train):
    return dict(**({"name": name} if name else {}), op=op, dtype=dtype, rows=rows, width=width, n_in=n_in, n_out=n_out, post=post, pre=pre,
                gate_rows=gate_rows, bias=bias, params=params, offset=offset, train=train)


def _cache(op, name, fmt, dtype, tokens, heads, dim, page, seqs, packed, padded):
    return dict(**({"name": name} if name else {}), op=op, fmt=fmt, dtype=dtype, tokens=tokens, heads=heads, dim=dim, page=page,
                seqs=seqs, packed=packed, padded=padded)


def listed():
    return [
        # one decoding step of eight sequences behind a block split over eight ranks: latency
        _norm("norm", "norm 8 ranks 8 rows", "bf16", 8, 4096, 8, 8, "none", "rms", 0, False, "bf16", 0.0, False),
        # a prefill chunk: partial outputs of eight ranks folded, normed on both sides, stored to all eight
        _norm("norm", "norm 8 ranks 2048 rows", "bf16", 2048, 8192, 8, 8, "rms", "rms", 2048, False, "f32", 0.0, False),
        # a conditioned model's layer: layer norms with biases, one gate row per sample, odd width, y kept for training
        _norm("norm", "norm samples odd", "f16", 4985, 1025, 2, 1, "layer", "layer", 997, True, "f16", 0.0, True),
        # fine-tuning on a few short rows, gradients of two ranks' copies
        _norm("grad", "grad 64 rows", "bf16", 64, 1024, 1, 2, "rms", "rms", 0, False, "bf16", 1.0, True),
        # the conditioned layer's backward in 32 bits, gradients to two ranks
        _norm("grad", "grad samples odd", "f32", 4985, 1025, 2, 1, "layer", "layer", 997, True, "f32", 0.0, True),
        # pre-training: a micro-batch's whole sequence, one gate per channel
        _norm("grad", "grad 16384 rows", "bf16", 16384, 8192, 1, 1, "rms", "rms", 16384, False, "f32", 0.0, True),
        # one decoding step of 64 sequences, keys and values of a rank's heads: latency
        _cache("write", "write 64 tokens e4m3", "f8e4m3", "bf16", 64, 8, 128, 16, 64, False, False),
        # a long prefill
        _cache("write", "write 65536 tokens i8", "i8", "f16", 65536, 8, 128, 64, 16, False, False),
        # odd heads and pages, tokens of padding among the others
        _cache("write", "write odd e5m2", "f8e5m2", "f32", 10007, 5, 72, 13, 7, False, True),
        # chunked prefill in four bits: the chunk is written and its sequences are read as decoding will see them
        _cache("append", "append 2048 tokens f4", "f4e2m1", "bf16", 2048, 8, 128, 32, 4, False, False),
        # histories handed over to another rank's layout, packed one after the other
        _cache("read", "read packed odd e4m3", "f8e4m3", "f32", 30011, 3, 80, 24, 11, True, False),
        # long contexts for attention over plain tensors
        _cache("read", "read 131072 tokens f4", "f4e2m1", "bf16", 131072, 8, 128, 64, 8, False, False),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["norm", "grad", "write", "append", "read"])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    if op in ("norm", "grad"):
        width = _log(rng, 64, 16384)
        if rng.random() < 0.5:
            width = max(64, width // 64 * 64)
        n_in, n_out = rng.choice([1, 2, 4, 8, rng.randint(1, 8)]), rng.choice([1, 2, 8, rng.randint(1, 8)])
        most = (1 << 29) // (width * BYTES[dtype] * (n_in + n_out + (4 if op == "grad" else 2)))
        rows = _log(rng, 1, max(1, min(32768, most)))
        gate_rows = rng.choice([0, 0, 1, rows, max(1, rows // rng.randint(2, 9))])
        post, pre = rng.choice([("none", "rms"), ("rms", "rms"), ("layer", "layer"), ("none", "layer"), ("rms", "none"), ("layer", "none")])
        return _norm(op, "", dtype, rows, width, n_in, n_out, post, pre, gate_rows, rng.random() < 0.3, rng.choice([dtype, "f32"]),
                     rng.choice([0.0, 0.0, 1.0]), op == "grad" or rng.random() < 0.3)
    heads, dim = rng.choice([1, 2, 4, 8, 16, rng.randint(1, 20)]), rng.choice([64, 128, 128, 256, rng.randint(16, 260)])
    most = (1 << 27) // (heads * dim * BYTES[dtype])
    tokens = _log(rng, 1, max(1, min(131072, most)))
    return _cache(op, "", rng.choice(sorted(FORMATS if op != "write" else [f for f in FORMATS if FORMATS[f]["bits"] == 8])), dtype,
                  tokens, heads, dim, rng.choice([1, 16, 16, 32, 64, rng.randint(2, 100)]), min(tokens, _log(rng, 1, 64)),
                  op == "read" and rng.random() < 0.5, rng.random() < 0.3)


# ---- inputs --------------------------------------------------------------------------------------------------------

def _rows_of_gate(case):
    return -(-case["rows"] // case["gate_rows"]) if case["gate_rows"] else 0


def _prepare_norm(case, gen):
    t, p = TYPES[case["dtype"]], TYPES[case["params"]]
    rows, width = case["rows"], case["width"]

    def normal(*shape, scale=1.0, mean=0.0, to=t):
        return (torch.randn(*shape, generator=gen, device="cuda") * scale + mean).to(to)

    s = dict(case=case, rows=rows, gate_rows=case["gate_rows"], post=case["post"], pre=case["pre"], offset=case["offset"],
             post_eps=1e-6, pre_eps=1e-6, residual_scale=1.0, block_scale=0.5)
    # a few channels of the residual stream carry far larger values than the others, as trained models' do
    channel = torch.ones(width, device="cuda")
    channel[torch.randint(0, width, (max(1, width // 200),), generator=gen, device="cuda")] = 20.0
    mean = 0.0 if case["offset"] else 1.0
    for side in ("post", "pre"):
        on = case[side] != "none"
        s[side + "_weight"] = normal(width, scale=0.2, mean=mean, to=p) if on else None
        s[side + "_bias"] = normal(width, scale=0.1, to=p) if on and case["bias"] else None
    s["gate"] = normal(_rows_of_gate(case), width, scale=0.5, mean=0.5, to=p) if case["gate_rows"] else None
    if case["op"] == "norm":
        s["parts"] = normal(case["n_in"], rows, width, scale=case["n_in"] ** -0.5)
        s["ins"] = list(s["parts"])
        s["residual"] = (normal(rows, width, to=torch.float32) * channel).to(t)
        s["residual_out"] = torch.empty(rows, width, dtype=t, device="cuda")
        s["folded"] = torch.empty(rows, width, dtype=t, device="cuda") if case["train"] else None
        s["copies"] = torch.empty(case["n_out"], rows, width, dtype=t, device="cuda")
        s["outs"] = list(s["copies"])
    else:
        s["folded"] = normal(rows, width)
        s["residual_out"] = (normal(rows, width, to=torch.float32) * channel).to(t)
        s["grad_copies"] = normal(case["n_out"], rows, width, scale=0.1)
        s["grad_outs"] = list(s["grad_copies"])
        s["grad_residual_out"] = normal(rows, width, scale=0.1)
        s["grad_parts"] = torch.empty(case["n_in"], rows, width, dtype=t, device="cuda")
        s["grad_ins"] = list(s["grad_parts"])
        s["grad_residual"] = torch.empty(rows, width, dtype=t, device="cuda")
        for name in ("gate", "post_weight", "post_bias", "pre_weight", "pre_bias"):
            s["grad_" + name] = None if s[name] is None else torch.empty_like(s[name])
    return s


def _prepare_cache(case, gen):
    fmt, heads, dim, page, tokens, seqs = case["fmt"], case["heads"], case["dim"], case["page"], case["tokens"], case["seqs"]
    bits = FORMATS[fmt]["bits"]
    s = dict(case=case, fmt=fmt, heads=heads, dim=dim, page=page, tokens=tokens, seqs=seqs)
    # lengths: uneven shares of the tokens, at least one each, the same for every seed (the pages' places are not)
    share = torch.arange(seqs, device="cuda", dtype=torch.float64) * 0.618 % 1 + 0.2
    lengths = 1 + ((tokens - seqs) * share / share.sum()).floor().long()
    lengths[0] += tokens - lengths.sum()
    if case["op"] == "write" and tokens == seqs:  # decoding: every sequence adds one token to a history
        positions = torch.arange(seqs, device="cuda") * 397 % 1024
        pages_of = positions // page + 1
    else:
        pages_of = (lengths + page - 1) // page
    per_seq = int(pages_of.max())
    pages = int(pages_of.sum()) + 3
    order = torch.randperm(pages, generator=gen, device="cuda")
    first = pages_of.cumsum(0) - pages_of
    column = torch.arange(per_seq, device="cuda")
    table = torch.where(column < pages_of[:, None], order[(first[:, None] + column).clamp(max=pages - 1)], -1)
    s["page_table"], s["lengths"] = table.to(torch.int32).contiguous(), lengths.to(torch.int32)
    seq = torch.repeat_interleave(torch.arange(seqs, device="cuda"), lengths)
    start = lengths.cumsum(0) - lengths
    pos = torch.arange(tokens, device="cuda") - start[seq]
    if case["op"] == "write" and tokens == seqs:
        seq, pos = torch.arange(seqs, device="cuda"), positions
    slots = table[seq, pos // page].long() * page + pos % page
    if case["padded"]:
        slots = torch.where(torch.rand(tokens, generator=gen, device="cuda") < 0.1, -1, slots)
    s["slots"], s["pages"], s["max_len"] = slots, pages, int(lengths.max())
    s["row_start"] = start if case["packed"] else None
    # keys and values: each a tensor of codes and one of scales, pages x tokens of a page x heads x bytes of a head
    row, blocks = (dim * bits + 7) // 8, -(-dim // BLOCK)
    shape = (2, pages, page, heads)
    if fmt in ("f8e4m3", "f8e5m2"):
        codes = torch.randn(*shape, row, generator=gen, device="cuda").mul_(FORMATS[fmt]["top"] / 6).clamp_(-FORMATS[fmt]["top"], FORMATS[fmt]["top"])
        codes = codes.to(torch.float8_e4m3fn if fmt == "f8e4m3" else torch.float8_e5m2).view(torch.uint8)
    elif fmt == "i8":
        codes = torch.randint(-127, 128, (*shape, row), generator=gen, device="cuda", dtype=torch.int8).view(torch.uint8)
    else:
        codes = torch.randint(0, 256, (*shape, row), generator=gen, device="cuda", dtype=torch.uint8)
    s["codes"] = codes
    s["powers"] = torch.tensor([2.0 ** i for i in range(-127, 128)], device="cuda")
    s["f4_values"] = torch.tensor(F4_VALUES, device="cuda")
    s["scales"] = torch.randint(124, 131, (*shape, blocks), generator=gen, device="cuda", dtype=torch.uint8) - FORMATS[fmt]["emax"]
    t = TYPES[case["dtype"]]
    if case["op"] != "read":
        # heads differ in size, and keys have channels that stand out
        size = torch.exp(torch.randn(2, 1, heads, 1, generator=gen, device="cuda")) * torch.exp(
            0.7 * torch.randn(2, 1, 1, dim, generator=gen, device="cuda"))
        s["source"] = (torch.randn(2, tokens, heads, dim, generator=gen, device="cuda") * size).to(t)
        s["sources"] = list(s["source"])
    if case["op"] != "write":
        shape = (2, tokens, heads, dim) if case["packed"] else (2, seqs, s["max_len"], heads, dim)
        s["out"] = torch.full(shape, 7.0, dtype=t, device="cuda")  # what stands behind a sequence's end is left as it is
        s["outs"] = list(s["out"])
    return s


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    s = (_prepare_norm if case["op"] in ("norm", "grad") else _prepare_cache)(case, gen)
    s["stream"] = torch.cuda.current_stream().cuda_stream
    if own:
        from pccl_amd import hip
        if case["op"] in ("norm", "grad"):
            s["layer"] = hip.FoldNorm(case["dtype"], case["width"], post=s["post"], pre=s["pre"], param_dtype=case["params"],
                                      post_weight=s["post_weight"], post_bias=s["post_bias"], pre_weight=s["pre_weight"],
                                      pre_bias=s["pre_bias"], post_eps=s["post_eps"], pre_eps=s["pre_eps"], weight_offset=s["offset"],
                                      residual_scale=s["residual_scale"], block_scale=s["block_scale"])
            if case["op"] == "grad":
                need = s["layer"].workspace_bytes(case["rows"], case["gate_rows"])
                s["workspace"] = torch.empty(max(need, 16), dtype=torch.uint8, device="cuda")
        else:
            s["cache"] = hip.Cache(case["fmt"], case["heads"], case["dim"], case["page"], s["pages"], list(s["codes"]), list(s["scales"]))
    return s


# ---- the framework's operators -------------------------------------------------------------------------------------

def _own(s):
    op = s["case"]["op"]
    if op == "norm":
        s["layer"].forward(s["ins"], s["outs"], s["rows"], residual=s["residual"], residual_out=s["residual_out"], folded=s["folded"],
                           gate=s["gate"], gate_rows=s["gate_rows"], stream=s["stream"])
        return {"residual": s["residual_out"], "folded": s["folded"], "outs": s["copies"]}
    if op == "grad":
        s["layer"].backward([s["folded"]], s["grad_outs"], s["grad_ins"], s["rows"], residual_out=s["residual_out"],
                            grad_residual_out=s["grad_residual_out"], grad_residual=s["grad_residual"], gate=s["gate"],
                            gate_rows=s["gate_rows"], grad_gate=s["grad_gate"], grad_post_weight=s["grad_post_weight"],
                            grad_post_bias=s["grad_post_bias"], grad_pre_weight=s["grad_pre_weight"], grad_pre_bias=s["grad_pre_bias"],
                            workspace=s["workspace"], stream=s["stream"])
        return _grads(s, s["grad_parts"], s["grad_residual"], s["grad_gate"], s["grad_post_weight"], s["grad_post_bias"],
                      s["grad_pre_weight"], s["grad_pre_bias"])
    t = s["case"]["dtype"]
    if op != "read":
        s["cache"].write(t, s["sources"], s["slots"], s["tokens"], stream=s["stream"])
    if op == "write":
        return _held(s["fmt"], s["codes"], s["scales"])
    if s["row_start"] is None:
        s["cache"].read(t, s["outs"], s["page_table"], s["lengths"], s["seqs"], s["max_len"], stream=s["stream"])
    else:
        s["cache"].read(t, s["outs"], s["page_table"], s["lengths"], s["seqs"], s["max_len"], row_start=s["row_start"],
                        out_rows=s["tokens"], stream=s["stream"])
    return s["out"]


def _grads(s, parts, residual, gate, post_weight, post_bias, pre_weight, pre_bias):
    return {"ins": parts, "residual": residual, "gate": gate, "post_weight": post_weight, "post_bias": post_bias,
            "pre_weight": pre_weight, "pre_bias": pre_bias}


def _held(fmt, codes, scales):
    """8-bit codes and scales as the values they stand for."""
    kind = {"f8e4m3": torch.float8_e4m3fn, "f8e5m2": torch.float8_e5m2, "i8": torch.int8}[fmt]
    return {"codes": codes.view(kind), "scales": scales.view(torch.float8_e8m0fnu)}


# ---- the plain forms -----------------------------------------------------------------------------------------------

def _normed(v, kind, weight, bias, offset, eps):
    """(the norm of v's rows, v standardised, one over its spread)"""
    if kind == "none":
        return v, v, None
    v = v - v.mean(-1, keepdim=True) if kind == "layer" else v
    rstd = 1 / torch.sqrt((v * v).mean(-1, keepdim=True) + eps)
    hat = v * rstd
    out = hat if weight is None else hat * (weight.float() + offset)
    return out if bias is None else out + bias.float(), hat, rstd


def _back(d, kind, hat, rstd, weight, offset):
    """The gradient of a norm's input from that of its output."""
    if kind == "none":
        return d
    d = d if weight is None else d * (weight.float() + offset)
    along = hat * (d * hat).mean(-1, keepdim=True)
    return rstd * (d - along - d.mean(-1, keepdim=True) if kind == "layer" else d - along)


def _gate_of_row(s):
    """Each row's gate, or None."""
    if s["gate"] is None:
        return None
    rows = torch.arange(s["rows"], device="cuda") // s["gate_rows"]
    return s["gate"].float()[rows] if s["gate"].shape[0] > 1 else s["gate"].float()


def _plain_norm(s):
    t = TYPES[s["case"]["dtype"]]
    y = s["parts"].float().sum(0)
    n, _, _ = _normed(y, s["post"], s["post_weight"], s["post_bias"], s["offset"], s["post_eps"])
    gate = _gate_of_row(s)
    n = n * s["block_scale"] if gate is None else n * gate * s["block_scale"]
    r = s["residual"].float() * s["residual_scale"] + n
    h, _, _ = _normed(r, s["pre"], s["pre_weight"], s["pre_bias"], s["offset"], s["pre_eps"])
    return {"residual": r.to(t), "folded": y.to(t) if s["case"]["train"] else None, "outs": h.to(t).expand(s["case"]["n_out"], -1, -1).contiguous()}


def _plain_grad(s):
    t, p = TYPES[s["case"]["dtype"]], TYPES[s["case"]["params"]]
    n, y_hat, y_rstd = _normed(s["folded"].float(), s["post"], s["post_weight"], s["post_bias"], s["offset"], s["post_eps"])
    _, r_hat, r_rstd = _normed(s["residual_out"].float(), s["pre"], s["pre_weight"], s["pre_bias"], s["offset"], s["pre_eps"])
    dh = s["grad_copies"].float().sum(0)
    dr = s["grad_residual_out"].float() + _back(dh, s["pre"], r_hat, r_rstd, s["pre_weight"], s["offset"])
    gate = _gate_of_row(s)
    dn = dr * s["block_scale"] if gate is None else dr * gate * s["block_scale"]
    dy = _back(dn, s["post"], y_hat, y_rstd, s["post_weight"], s["offset"])
    dgate = None
    if gate is not None:
        each = dr * n * s["block_scale"]
        full = torch.nn.functional.pad(each, (0, 0, 0, s["gate"].shape[0] * s["gate_rows"] - s["rows"]))
        dgate = full.view(s["gate"].shape[0], s["gate_rows"], -1).sum(1).to(p)
    return _grads(s, dy.to(t).expand(s["case"]["n_in"], -1, -1).contiguous(), (dr * s["residual_scale"]).to(t), dgate,
                  None if s["post_weight"] is None else (dn * y_hat).sum(0).to(p), None if s["post_bias"] is None else dn.sum(0).to(p),
                  None if s["pre_weight"] is None else (dh * r_hat).sum(0).to(p), None if s["pre_bias"] is None else dh.sum(0).to(p))


def _power_of_two(s, k):
    """2^k for whole k in [-127, 127], exactly: from a list, for a device's pow may be a unit off."""
    return s["powers"][k.long() + 127]


def _plain_write(s):
    f, dim = FORMATS[s["fmt"]], s["dim"]
    x = torch.nn.functional.pad(s["source"].float(), (0, -dim % BLOCK)).unflatten(-1, (-1, BLOCK))
    most = x.abs().amax(-1, keepdim=True)
    fine = torch.isfinite(most)
    mantissa, exponent = torch.frexp(torch.where(fine, most, 0.0))
    k = exponent - 1 - f["emax"] + (2 * mantissa * 2.0 ** f["emax"] > f["top"])
    k = torch.where(most == 0, -127, k).clamp(-127, 127)
    v = torch.where(fine, x, 0.0) * _power_of_two(s, -k)  # a power of two: no rounding
    step = _power_of_two(s, (torch.frexp(v)[1] - 1).clamp(min=f["emin"]) - f["mbits"])
    v = (torch.round(v / step) * step).clamp(-f["top"], f["top"])  # to the nearest, ties to even
    v = v.flatten(-2)[..., :dim]
    if s["fmt"] == "i8":
        codes = (v * 64).to(torch.int8).view(torch.uint8)
    elif f["bits"] == 8:
        codes = v.to(torch.float8_e4m3fn if s["fmt"] == "f8e4m3" else torch.float8_e5m2).view(torch.uint8)
    else:
        a = v.abs()
        code = (2 * a - (a - 2).clamp(min=0) - (a - 4).clamp(min=0) / 2).to(torch.uint8) + 8 * torch.signbit(v).to(torch.uint8)
        code = torch.nn.functional.pad(code, (0, dim % 2))
        codes = code[..., 0::2] + 16 * code[..., 1::2]
    scales = torch.where(fine, k + 127, 255).to(torch.uint8).squeeze(-1)
    slots = s["slots"]
    if s["case"]["padded"]:  # slots below zero name tokens that are not kept
        named = slots >= 0
        slots, codes, scales = slots[named], codes[:, named], scales[:, named]
    s["codes"].flatten(1, 2)[:, slots] = codes
    s["scales"].flatten(1, 2)[:, slots] = scales


def _plain_read(s):
    f, dim, t = FORMATS[s["fmt"]], s["dim"], TYPES[s["case"]["dtype"]]
    if s["row_start"] is None:
        pos = torch.arange(s["max_len"], device="cuda").expand(s["seqs"], -1)
        seq = torch.arange(s["seqs"], device="cuda")[:, None].expand(-1, s["max_len"])
    else:
        row = torch.arange(s["tokens"], device="cuda")
        seq = torch.searchsorted(s["row_start"], row, right=True) - 1
        pos = row - s["row_start"][seq]
    within = pos < s["lengths"][seq]
    at = s["page_table"][seq, torch.where(within, pos // s["page"], 0)].long().clamp(min=0)
    codes, scales = s["codes"][:, at, pos % s["page"]], s["scales"][:, at, pos % s["page"]]
    if s["fmt"] == "i8":
        v = codes.view(torch.int8).float() / 64
    elif f["bits"] == 8:
        v = codes.view(torch.float8_e4m3fn if s["fmt"] == "f8e4m3" else torch.float8_e5m2).float()
    else:
        v = torch.stack([s["f4_values"][(codes & 15).long()], s["f4_values"][(codes >> 4).long()]], -1).flatten(-2)[..., :dim]
    scale = torch.where(scales == 255, math.nan, _power_of_two(s, scales.clamp(max=254).int() - 127))
    v = (v * scale.repeat_interleave(BLOCK, -1)[..., :dim]).to(t)
    s["out"].copy_(torch.where(within[..., None, None], v, s["out"]))
    return s["out"]


def _plain(s):
    op = s["case"]["op"]
    if op == "norm":
        return _plain_norm(s)
    if op == "grad":
        return _plain_grad(s)
    if op != "read":
        _plain_write(s)
    return _held(s["fmt"], s["codes"], s["scales"]) if op == "write" else _plain_read(s)


def run(state):
    return _own(state) if own else _plain(state)


# ---- what a pass cannot do without ---------------------------------------------------------------------------------

def work(case):
    if case["op"] in ("norm", "grad"):
        n, size, p = case["rows"] * case["width"], BYTES[case["dtype"]], BYTES[case["params"]]
        vectors = sum((case[side] != "none") * (2 if case["bias"] else 1) for side in ("post", "pre")) + _rows_of_gate(case)
        if case["op"] == "norm":
            return {"bytes": n * size * (case["n_in"] + 2 + case["n_out"] + case["train"]) + vectors * case["width"] * p,
                    "flops": n * (case["n_in"] + 12)}
        return {"bytes": n * size * (case["n_out"] + 4 + case["n_in"]) + 2 * vectors * case["width"] * p, "flops": n * (case["n_out"] + 30)}
    n = 2 * case["tokens"] * case["heads"] * case["dim"]
    held = 2 * case["tokens"] * case["heads"] * ((case["dim"] * FORMATS[case["fmt"]]["bits"] + 7) // 8 + -(-case["dim"] // BLOCK))
    once = n * BYTES[case["dtype"]] + held
    return {"bytes": once * (2 if case["op"] == "append" else 1), "flops": 3 * n * (2 if case["op"] == "append" else 1)}


# ---- the definition in 64 bits -------------------------------------------------------------------------------------

def _exact_layer(v, kind, weight, bias, offset, eps):
    if kind == "none":
        return v
    width = v.shape[-1]
    mean = v.sum(-1, keepdim=True) / width if kind == "layer" else 0.0
    spread = ((v - mean) ** 2).sum(-1, keepdim=True) / width
    out = (v - mean) * (spread + eps) ** -0.5
    if weight is not None:
        out = out * (weight + offset)
    return out if bias is None else out + bias


def _exact_norm(s):
    case, rows = s["case"], s["rows"]
    leaf = {k: s[k].double() for k in ("gate", "post_weight", "post_bias", "pre_weight", "pre_bias") if s[k] is not None}

    def chain(y, x, p):
        n = _exact_layer(y, s["post"], p.get("post_weight"), p.get("post_bias"), s["offset"], s["post_eps"])
        if "gate" in p:
            n = n * torch.repeat_interleave(p["gate"], s["gate_rows"], 0)[:rows]
        r = s["residual_scale"] * x + s["block_scale"] * n
        return r, lambda r: _exact_layer(r, s["pre"], p.get("pre_weight"), p.get("pre_bias"), s["offset"], s["pre_eps"])

    if case["op"] == "norm":
        y = s["parts"].double().sum(0)
        r, after = chain(y, s["residual"].double(), leaf)
        return {"residual": r, "folded": y if case["train"] else None, "outs": torch.stack([after(r)] * case["n_out"])}
    # the chain is cut at r, whose rounded value the backward pass is given
    leaf = {k: v.requires_grad_() for k, v in leaf.items()}
    y = s["folded"].double().requires_grad_()
    x = torch.zeros_like(y).requires_grad_()
    r, after = chain(y, x, leaf)
    r_given = s["residual_out"].double().requires_grad_()
    h = after(r_given)
    names = [k for k in leaf if k.startswith("pre_")]
    got = torch.autograd.grad(h, [r_given] + [leaf[k] for k in names], s["grad_copies"].double().sum(0))
    found = dict(zip(names, got[1:]))
    names = [k for k in leaf if not k.startswith("pre_")]
    got = torch.autograd.grad(r, [y, x] + [leaf[k] for k in names], got[0] + s["grad_residual_out"].double())
    found |= dict(zip(names, got[2:]))
    rest = (found.get(k) for k in ("gate", "post_weight", "post_bias", "pre_weight", "pre_bias"))
    return _grads(s, torch.stack([got[0]] * case["n_in"]), got[1], *rest)


def _values_of(fmt):
    """Every finite value of a format, by code, in 64 bits."""
    if fmt == "i8":
        return [(c - 256 if c > 127 else c) / 64 for c in range(256)]
    e, m = {"f8e4m3": (4, 3), "f8e5m2": (5, 2), "f4e2m1": (2, 1)}[fmt]
    bias, found = 2 ** (e - 1) - 1, []
    for c in range(2 ** (1 + e + m)):
        exponent, fraction = (c >> m) & (2 ** e - 1), c & (2 ** m - 1)
        v = (fraction / 2 ** m) * 2.0 ** (1 - bias) if exponent == 0 else (1 + fraction / 2 ** m) * 2.0 ** (exponent - bias)
        if fmt == "f8e5m2" and exponent == 31:
            v = math.inf if fraction == 0 else math.nan
        if fmt == "f8e4m3" and exponent == 15 and fraction == 7:
            v = math.nan
        found.append(-v if c >> (e + m) else v)
    return found


def _exact_scale(k):
    """2^k in 64 bits, exactly."""
    return torch.tensor([math.ldexp(1.0, i) for i in range(-130, 131)], dtype=torch.float64, device="cuda")[k.long() + 130]


def _exact_coded(s):
    """(values of the codes without their scale, scale exponents) of the source's blocks, from the nearest entry of the format's list."""
    grid = sorted({abs(v) for v in _values_of(s["fmt"]) if math.isfinite(v) and abs(v) <= FORMATS[s["fmt"]]["top"]})
    top, dim = grid[-1], s["dim"]
    x = s["source"].double()
    x = torch.cat([x, x.new_zeros(*x.shape[:-1], -dim % BLOCK)], -1).reshape(*x.shape[:-1], -1, BLOCK)
    most = x.abs().max(-1).values
    k = torch.ceil(torch.log2(most.clamp(min=1e-300) / top)).clamp(-127, 127)
    k = torch.where((most <= top * _exact_scale(k - 1)) & (k > -127), k - 1, k)
    k = torch.where((most > top * _exact_scale(k)) & (k < 127), k + 1, k)
    g = torch.tensor(grid, dtype=torch.float64, device="cuda")
    between = (g[1:] + g[:-1]) / 2
    a = x.abs() / _exact_scale(k)[..., None]
    low, high = torch.searchsorted(between, a), torch.searchsorted(between, a, right=True)  # they differ at a tie: the even one
    v = g[torch.where(low % 2 == 0, low, high)] * torch.where(torch.signbit(x), -1.0, 1.0)
    return v.flatten(-2)[..., :dim], k


def _exact_cache(s):
    case, dim = s["case"], s["dim"]
    values = torch.tensor(_values_of(s["fmt"]), dtype=torch.float64, device="cuda")
    codes = s["codes"].long()
    if s["fmt"] == "f4e2m1":
        codes = torch.stack([codes % 16, codes // 16], -1).flatten(-2)[..., :dim]
    held, scale = values[codes].flatten(1, 2), s["scales"].double().flatten(1, 2) - 127
    if case["op"] != "read":
        v, k = _exact_coded(s)
        named = s["slots"] >= 0
        held[:, s["slots"][named]], scale[:, s["slots"][named]] = v[:, named], k[:, named]
    if case["op"] == "write":
        shape = s["codes"].shape[:3]
        held = held * 64 if s["fmt"] == "i8" else held  # (returned as whole numbers)
        return {"codes": held.unflatten(1, shape[1:]), "scales": _exact_scale(scale).unflatten(1, shape[1:])}
    whole = held * torch.repeat_interleave(_exact_scale(scale), BLOCK, -1)[..., :dim]
    out = s["out"].double()
    for i, n in enumerate(s["lengths"].tolist()):
        pos = torch.arange(n, device="cuda")
        rows = whole[:, s["page_table"][i].long()[pos // s["page"]] * s["page"] + pos % s["page"]]
        if case["packed"]:
            first = int(s["row_start"][i])
            out[:, first:first + n] = rows
        else:
            out[:, i, :n] = rows
    return out


def exact(case, seed):
    s = prepare(case, seed)
    return _exact_norm(s) if case["op"] in ("norm", "grad") else _exact_cache(s)
