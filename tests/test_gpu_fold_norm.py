"""pccl_hip_fold_norm and its backward pass against the restatement in 64 bits of norm_reference.py, whose bounds are the
tolerances; widths around every edge of a pack, a wavefront and a team, odd strides and addresses, guard bands."""
import random

import pytest

import norm_reference as ref

pytestmark = pytest.mark.gpu

TYPES = [("f32", "f32"), ("bf16", "bf16"), ("bf16", "f32"), ("f16", "f16"), ("f16", "f32")]
KINDS = [("none", "rms"), ("rms", "rms"), ("layer", "layer"), ("rms", "layer"), ("layer", "none"), ("none", "none"), ("rms", "none"), ("none", "layer")]


class Rows:
    """rows x width elements `stride` apart on the device, `shift` elements behind a 256-byte boundary, in a band of a pattern."""

    def __init__(self, torch, dtype, rows, width, stride=None, shift=0, src=None):
        self.t = ref.TYPES[dtype]
        self.stride = width if stride is None else stride
        size = torch.finfo(self.t).bits // 8
        pad = 64
        self.raw = torch.full((2 * pad + shift + max(0, rows - 1) * self.stride + width,), -7.0, dtype=self.t, device="cuda")
        self.view = self.raw.as_strided((rows, width), (self.stride, 1), pad + shift)
        self.addr = self.raw.data_ptr() + (pad + shift) * size
        self.torch = torch
        if src is not None:
            self.view.copy_(src)

    def data_ptr(self):
        return self.addr

    def get(self):
        return self.view.double().cpu()

    def band_is_whole(self):
        """Nothing between or around the rows was written."""
        left = self.raw.clone()
        left.as_strided(self.view.shape, self.view.stride(), self.view.storage_offset()).fill_(-7.0)
        return bool((left == -7.0).all())


def close(got, want, dtype, what):
    value, bound = want
    off = (got - value).abs()
    allowed = bound + ref.rounding(dtype, value)
    bad = ~(off <= allowed)
    assert not bool(bad.any()), "%s: %d of %d beyond the bound, worst %.3g of %.3g" % (
        what, int(bad.sum()), bad.numel(), float((off / allowed).max()), float(allowed.max()))


def settings(torch, gen, dtype, params, width, post, pre, weights=True, biases=True, offset=0.0, a=1.0, c=1.0, gate_shape=None):
    """(parameters in 64 bits that are exact in their type, the same on the device)"""
    def vec(*shape, mean=0.0, scale=1.0):
        return (torch.randn(*shape, generator=gen) * scale + mean).to(ref.TYPES[params]).double()
    p = dict(post=post, pre=pre, weight_offset=offset, residual_scale=a, block_scale=c, post_eps=1e-5, pre_eps=1e-6)
    for side, kind in (("post", post), ("pre", pre)):
        p[side + "_weight"] = vec(width, mean=1.0 - offset, scale=0.3) if kind != "none" and weights else None
        p[side + "_bias"] = vec(width, scale=0.2) if kind != "none" and biases else None
    gate = None if gate_shape is None else vec(*gate_shape, mean=0.5)
    dev = {k: None if p[k] is None else p[k].to(ref.TYPES[params]).cuda() for k in ("post_weight", "post_bias", "pre_weight", "pre_bias")}
    return p, gate, dev


def layer(hip, dtype, params, width, p, dev):
    return hip.FoldNorm(dtype, width, param_dtype=params, **dev, **{k: v for k, v in p.items() if k not in dev})


def draws(seed, n):
    """Cases over all settings; widths at and around every edge."""
    rng = random.Random(seed)
    widths = [1, 2, 3, 4, 5, 7, 8, 9, 31, 63, 64, 65, 72, 127, 500, 511, 512, 513, 520, 1000, 1023, 1024, 1025, 1032, 2041, 2047, 2048, 2049,
              3000, 4095, 4096, 4097, 4100, 5003, 8190, 8192, 8193, 8200, 12289, 16376, 16383, 16384]
    for k in range(n):
        width = widths[k % len(widths)]
        rows = rng.choice([1, 2, 3, 4, 5, 9, 37, 130]) if width < 5000 else rng.choice([1, 2, 5, 17])
        gate = rng.choice(["none", "none", "one", "row", "some"])
        gate_rows = {"none": 0, "one": rows + rng.randint(0, 3), "row": 1, "some": max(1, rows // 3)}[gate]
        yield dict(types=TYPES[k % 5], kinds=KINDS[rng.randrange(8)], width=width, rows=rows, n_in=rng.randint(1, 8), n_out=rng.randint(0, 8),
                   gate_rows=gate_rows, weights=rng.random() < 0.8, biases=rng.random() < 0.5, offset=rng.choice([0.0, 1.0]),
                   a=rng.choice([1.0, 0.75, -2.0]), c=rng.choice([1.0, 0.5]), residual=rng.random() < 0.8, pad=rng.choice([0, 0, 1, 3, 8, 13]),
                   shift=rng.choice([0, 0, 1, 2, 5, 8]), seed=rng.randrange(1 << 30))


def name(c):
    return "%s-%s-%s-%s-w%d-r%d-i%d-o%d-g%d" % (*c["types"], *c["kinds"], c["width"], c["rows"], c["n_in"], c["n_out"], c["gate_rows"])


def values(torch, gen, dtype, *shape, scale=1.0):
    return (torch.randn(*shape, generator=gen) * scale).to(ref.TYPES[dtype]).double()


def prepared(torch, c):
    gen = torch.Generator().manual_seed(c["seed"])
    rows, width, (dtype, params) = c["rows"], c["width"], c["types"]
    shape = (-(-rows // c["gate_rows"]), width) if c["gate_rows"] else None
    p, gate, dev = settings(torch, gen, dtype, params, width, *c["kinds"], c["weights"], c["biases"], c["offset"], c["a"], c["c"], shape)
    return gen, p, gate, dev


def put(torch, c, rows, src, k=0):
    return Rows(torch, c["types"][0], rows, c["width"], c["width"] + c["pad"], c["shift"] if k % 2 == 0 else 0, src)


@pytest.mark.parametrize("c", list(draws(11, 84)), ids=name)
def test_forward(hip, c):
    import torch
    gen, p, gate, dev = prepared(torch, c)
    dtype, params = c["types"]
    rows, width = c["rows"], c["width"]
    parts = values(torch, gen, dtype, c["n_in"], rows, width)
    x = values(torch, gen, dtype, rows, width, scale=2.0) if c["residual"] else None
    want = ref.forward(parts, x, gate, c["gate_rows"], p)
    ins = [put(torch, c, rows, parts[k], k) for k in range(c["n_in"])]
    d_x = None if x is None else put(torch, c, rows, x, 1)
    r, y = put(torch, c, rows, None), put(torch, c, rows, None, 1)
    outs = [put(torch, c, rows, None, k) for k in range(c["n_out"])]
    g = None if gate is None else Rows(torch, params, gate.shape[0], width, width + c["pad"], c["shift"], gate)
    stride = width + c["pad"]
    layer(hip, dtype, params, width, p, dev).forward(
        ins, outs, rows, residual=d_x, residual_out=r, folded=y, gate=g, gate_rows=c["gate_rows"], gate_stride=stride,
        stream=torch.cuda.current_stream().cuda_stream, in_stride=stride, residual_stride=stride, residual_out_stride=stride, folded_stride=stride,
        out_stride=stride)
    torch.cuda.synchronize()
    close(y.get(), want["folded"], dtype, "folded")
    close(r.get(), want["residual_out"], dtype, "residual_out")
    for o in outs:
        close(o.get(), want["outs"], dtype, "outs")
        assert torch.equal(o.get(), outs[0].get())
    for b in [r, y] + outs + ins:
        assert b.band_is_whole()


@pytest.mark.parametrize("c", list(draws(12, 84)), ids=name)
def test_backward(hip, c):
    import torch
    gen, p, gate, dev = prepared(torch, c)
    dtype, params = c["types"]
    rows, width, n_out = c["rows"], c["width"], c["n_out"]
    n_in = 1 if c["n_in"] % 2 else c["n_in"]  # y as kept, or the partial outputs again
    parts = values(torch, gen, dtype, n_in, rows, width)
    r = values(torch, gen, dtype, rows, width, scale=2.0)
    dh = values(torch, gen, dtype, n_out, rows, width) if n_out else None
    dr = values(torch, gen, dtype, rows, width) if c["residual"] else torch.zeros(rows, width, dtype=torch.float64)
    want = ref.backward(parts, r, dh, dr, gate, c["gate_rows"], p)
    stride = width + c["pad"]
    ins = [put(torch, c, rows, parts[k], k) for k in range(n_in)]
    d_r = put(torch, c, rows, r)
    d_dh = [put(torch, c, rows, dh[k], k) for k in range(n_out)]
    d_dr = put(torch, c, rows, dr, 1) if c["residual"] else None
    g = None if gate is None else Rows(torch, params, gate.shape[0], width, stride, c["shift"], gate)
    grad_ins = [put(torch, c, rows, None, k) for k in range(c["n_in"])]
    grad_x = put(torch, c, rows, None)
    grad_g = None if gate is None else Rows(torch, params, gate.shape[0], width, stride, c["shift"])
    grads = {"grad_" + k: None if v is None else Rows(torch, params, 1, width) for k, v in dev.items()}
    L = layer(hip, dtype, params, width, p, dev)
    need = L.workspace_bytes(rows, c["gate_rows"])
    ws = torch.full((need + 256,), 0x5A, dtype=torch.uint8, device="cuda")

    def call():
        L.backward(ins, d_dh, grad_ins, rows, residual_out=d_r, grad_residual_out=d_dr, grad_residual=grad_x, gate=g, gate_rows=c["gate_rows"],
                   grad_gate=grad_g, workspace=ws, workspace_bytes=need, stream=torch.cuda.current_stream().cuda_stream, in_stride=stride,
                   residual_out_stride=stride, gate_stride=stride, grad_out_stride=stride, grad_residual_out_stride=stride, grad_in_stride=stride,
                   grad_residual_stride=stride, grad_gate_stride=stride, **grads)
        torch.cuda.synchronize()

    call()
    assert bool((ws[need:] == 0x5A).all())
    close(grad_x.get(), want["grad_residual"], dtype, "grad_residual")
    for k, b in enumerate(grad_ins):
        close(b.get(), want["grad_ins"], dtype, "grad_ins")
        assert b.band_is_whole()
    if gate is not None:
        close(grad_g.get(), want["grad_gate"], params, "grad_gate")
        assert grad_g.band_is_whole()
    for k, b in grads.items():
        if b is not None:
            zero = torch.zeros(width, dtype=torch.float64)
            close(b.get()[0], want.get(k, (zero, zero)), params, k)
            assert b.band_is_whole()
    # the same call gives the same bits
    before = [b.raw.clone() for b in [grad_x] + grad_ins + [b for b in grads.values() if b is not None]]
    ws.fill_(0x33)
    call()
    for was, b in zip(before, [grad_x] + grad_ins + [b for b in grads.values() if b is not None]):
        assert torch.equal(was, b.raw)
