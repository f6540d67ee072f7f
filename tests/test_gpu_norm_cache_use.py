"""The norms around a block and the cache in blocks as programs use them: in place, on other streams, captured and replayed, from two
threads, with strides and offsets beyond 32 bits, with masked and padded rows, one behind the other in a layer's step together with
the library's folds and copies; gradients against differences."""
import threading

import pytest

import cache_reference as cref
import norm_reference as ref

pytestmark = pytest.mark.gpu


def params(torch, gen, width, dtype, post="rms", pre="rms", biases=False, **kw):
    t = ref.TYPES[dtype]
    p = dict(post=post, pre=pre, weight_offset=0.0, residual_scale=1.0, block_scale=0.5, post_eps=1e-6, pre_eps=1e-6, **kw)
    for side, kind in (("post", post), ("pre", pre)):
        p[side + "_weight"] = (1 + 0.2 * torch.randn(width, generator=gen)).to(t).double() if kind != "none" else None
        p[side + "_bias"] = (0.1 * torch.randn(width, generator=gen)).to(t).double() if biases and kind != "none" else None
    return p


def layer_of(hip, dtype, width, p):
    on_device = {k: None if p[k] is None else p[k].to(ref.TYPES[dtype]).cuda() for k in ("post_weight", "post_bias", "pre_weight", "pre_bias")}
    return hip.FoldNorm(dtype, width, **on_device, **{k: v for k, v in p.items() if k not in on_device})


def rows(torch, gen, dtype, *shape, scale=1.0):
    return (torch.randn(*shape, generator=gen) * scale).to(ref.TYPES[dtype])


def within(got, want, dtype, what):
    off, allowed = (got.double().cpu() - want[0]).abs(), want[1] + ref.rounding(dtype, want[0])
    assert bool((off <= allowed).all()), "%s: worst %.3g of its bound" % (what, float((off / allowed).max()))


@pytest.mark.parametrize("width", [64, 513, 1000, 4096, 9000])
def test_in_place(hip, width):
    """r over x, h over a partial output; in the backward dy over y, dx over the gradient from further on."""
    import torch
    gen = torch.Generator().manual_seed(1)
    n, dtype = 37, "bf16"
    p = params(torch, gen, width, dtype)
    parts, x = rows(torch, gen, dtype, 2, n, width), rows(torch, gen, dtype, n, width)
    want = ref.forward(parts.double(), x.double(), None, 0, p)
    L, d_parts, d_x = layer_of(hip, dtype, width, p), parts.cuda(), x.cuda()
    L.forward([d_parts[0], d_parts[1]], [d_parts[1]], n, residual=d_x, residual_out=d_x, folded=d_parts[0])
    torch.cuda.synchronize()
    within(d_parts[0], want["folded"], dtype, "folded")
    within(d_x, want["residual_out"], dtype, "residual_out")
    within(d_parts[1], want["outs"], dtype, "outs")
    y, r, dh, dr = (rows(torch, gen, dtype, n, width) for _ in range(4))
    want = ref.backward(y.double()[None], r.double(), dh.double()[None], dr.double(), None, 0, p)
    d_y, d_r, d_dh, d_dr = y.cuda(), r.cuda(), dh.cuda(), dr.cuda()
    L.backward([d_y], [d_dh], [d_y], n, residual_out=d_r, grad_residual_out=d_dr, grad_residual=d_dr)
    torch.cuda.synchronize()
    within(d_y, want["grad_ins"], dtype, "grad_ins")
    within(d_dr, want["grad_residual"], dtype, "grad_residual")


@pytest.mark.parametrize("dtype,kinds,width", [("f32", ("rms", "rms"), 24), ("f32", ("layer", "layer"), 700), ("f32", ("layer", "none"), 1300), ("f32", ("none", "layer"), 4100)])
def test_gradients_against_differences(hip, dtype, kinds, width):
    """A step of every input at once along a random direction, the loss differenced in 64 bits: the gradients' product with the
    direction.  Error: the square of the step (1e-4 of the inputs, which are of size 1) and the kernel's 2^-24 a term, far below 1e-5 of
    the sum of the terms' magnitudes."""
    import torch
    gen = torch.Generator().manual_seed(7)
    n, gate_rows = 11, 4
    p = params(torch, gen, width, dtype, *kinds, biases=True)
    groups = -(-n // gate_rows)
    gate = rows(torch, gen, dtype, groups, width).double()
    parts, x = rows(torch, gen, dtype, 1, n, width).double(), rows(torch, gen, dtype, n, width).double()
    dh, dr = rows(torch, gen, dtype, n, width).double(), rows(torch, gen, dtype, n, width).double()
    r = ref.forward(parts, x, gate, gate_rows, p)["residual_out"][0].float().double()  # as a forward pass in 32 bits leaves it
    names = [k for k in ("post_weight", "post_bias", "pre_weight", "pre_bias") if p[k] is not None]
    step = dict(parts=torch.randn(parts.shape, generator=gen).double(), x=torch.randn(x.shape, generator=gen).double(),
                gate=torch.randn(gate.shape, generator=gen).double(), **{k: torch.randn(width, generator=gen).double() for k in names})

    def loss(e):
        q = dict(p, **{k: p[k] + e * step[k] for k in names})
        f = ref.forward(parts + e * step["parts"], x + e * step["x"], gate + e * step["gate"], gate_rows, q)
        return float((f["outs"][0] * dh).sum() + (f["residual_out"][0] * dr).sum())

    e = 1e-4
    slope = (loss(e) - loss(-e)) / (2 * e)
    L = layer_of(hip, dtype, width, p)
    dev = lambda v: v.to(ref.TYPES[dtype]).cuda()  # noqa: E731
    got = {k: torch.zeros_like(dev(v)) for k, v in (("parts", parts[0]), ("x", x), ("gate", gate))} | {k: torch.zeros(width, device="cuda") for k in names}
    L.backward([dev(parts[0])], [dev(dh)], [got["parts"]], n, residual_out=dev(r), grad_residual_out=dev(dr), grad_residual=got["x"], gate=dev(gate),
               gate_rows=gate_rows, grad_gate=got["gate"], workspace=torch.zeros(L.workspace_bytes(n, gate_rows), dtype=torch.uint8, device="cuda"),
               **{"grad_" + k: got[k] for k in names})
    torch.cuda.synchronize()
    terms = torch.cat([(got[k].double().cpu().view(-1) * step[k].view(-1)) for k in got])
    assert abs(float(terms.sum()) - slope) <= 1e-5 * float(terms.abs().sum())


def test_rows_beyond_one_launch(hip):
    """More rows than one launch's grid takes (2^21)."""
    import torch
    n, width = (1 << 21) + 5, 8
    gen = torch.Generator().manual_seed(3)
    p = params(torch, gen, width, "bf16")
    L = layer_of(hip, "bf16", width, p)
    some = rows(torch, gen, "bf16", 1021, width)
    y = some.repeat(n // 1021 + 1, 1)[:n].cuda()
    gate = torch.ones(2, width, dtype=torch.bfloat16, device="cuda")
    gate[1] = 2.0  # rows of the second launch and a few of the first
    gate_rows = (1 << 21) - 3
    out, r = torch.zeros_like(y), torch.zeros_like(y)
    L.forward([y], [out], n, residual_out=r, gate=gate, gate_rows=gate_rows)
    torch.cuda.synchronize()
    for lo in (0, gate_rows - 7, (1 << 21) - 20, n - 20):
        part = y[lo:lo + 20].cpu().double()
        g = torch.where(torch.arange(lo, lo + 20)[:, None] < gate_rows, 1.0, 2.0).expand(-1, width).double()[:part.shape[0]]
        want = ref.forward(part[None], None, g, 1, p)
        within(r[lo:lo + 20], want["residual_out"], "bf16", "rows from %d" % lo)
        within(out[lo:lo + 20], want["outs"], "bf16", "rows from %d" % lo)


def test_row_offsets_beyond_32_bits(hip):
    """Rows so far apart that their offsets pass 2^32 bytes, forward and backward."""
    import torch
    width, n, stride = 96, 3, (1 << 30) + 40  # elements: 2 GiB apart
    gen = torch.Generator().manual_seed(4)
    p = params(torch, gen, width, "bf16")
    L = layer_of(hip, "bf16", width, p)
    y, x, dh, dr = (rows(torch, gen, "bf16", n, width) for _ in range(4))
    big = torch.empty((n - 1) * stride + 4096, dtype=torch.bfloat16, device="cuda")  # 4 GiB: y, x, r and h take turns in each of its rows
    view = lambda at: big.as_strided((n, width), (stride, 1), at)  # noqa: E731
    v_y, v_x, v_h, v_dh, v_dr = view(0), view(128), view(256), view(384), view(512)
    for v, s in ((v_y, y), (v_x, x), (v_dh, dh), (v_dr, dr)):
        v.copy_(s)
    at = lambda v: big.data_ptr() + 2 * v.storage_offset()  # noqa: E731
    L.forward([at(v_y)], [at(v_h)], n, residual=at(v_x), residual_out=at(v_x), in_stride=stride, out_stride=stride, residual_stride=stride,
              residual_out_stride=stride)
    torch.cuda.synchronize()
    want = ref.forward(y.double()[None], x.double(), None, 0, p)
    within(v_h, want["outs"], "bf16", "h")
    within(v_x, want["residual_out"], "bf16", "r")
    v_x.copy_(x)
    L.backward([at(v_y)], [at(v_dh)], [at(v_y)], n, residual_out=at(v_x), grad_residual_out=at(v_dr), grad_residual=at(v_dr), in_stride=stride,
               grad_out_stride=stride, grad_in_stride=stride, residual_out_stride=stride, grad_residual_out_stride=stride, grad_residual_stride=stride)
    torch.cuda.synchronize()
    want = ref.backward(y.double()[None], x.double(), dh.double()[None], dr.double(), None, 0, p)
    within(v_y, want["grad_ins"], "bf16", "dy")
    within(v_dr, want["grad_residual"], "bf16", "dx")


def test_zero_constant_and_infinite_rows(hip):
    """Rows of zeros and constant rows are divided by the root of eps; a NaN or an infinity stays in its row."""
    import torch
    for kinds in (("rms", "rms"), ("layer", "layer")):
        for dtype in ("f32", "bf16", "f16"):
            width, n = 700, 8
            gen = torch.Generator().manual_seed(5)
            p = params(torch, gen, width, dtype, *kinds)
            y = rows(torch, gen, dtype, n, width)
            y[0], y[1], y[2] = 0, 3.0, -0.0
            y[4, 17], y[5, 650], y[6, 3] = float("nan"), float("inf"), torch.finfo(y.dtype).min if dtype == "f16" else -1e15
            L = layer_of(hip, dtype, width, p)
            out, d_y = torch.zeros(n, width, dtype=y.dtype, device="cuda"), y.cuda()
            L.forward([d_y], [out], n, residual=torch.zeros_like(out))
            torch.cuda.synchronize()
            want = ref.forward(y.double()[None], None, None, 0, p)["outs"]
            fine = [0, 1, 2, 3, 6, 7]
            assert not bool(torch.isfinite(out[4]).any()) and bool(torch.isnan(out[5]).any())
            within(out[fine], (want[0][fine], want[1][fine]), dtype, "%s %s" % (kinds, dtype))


@pytest.mark.parametrize("width", [40, 700, 9000])
def test_tiny_eps(hip, width):
    """eps near the smallest it may be: rows of zeros have gradients of zero and 1 / sqrt(eps), not NaN."""
    import torch
    n = 5
    gen = torch.Generator().manual_seed(6)
    p = params(torch, gen, width, "f32")
    p["post_eps"] = p["pre_eps"] = 1e-37
    L = layer_of(hip, "f32", width, p)
    y, r, dh = (rows(torch, gen, "f32", n, width) for _ in range(3))
    y[1], r[2], r[3], dh[2], dh[3] = 0, 0, 0, 0, dh[3] * 1e-20
    new = lambda: torch.zeros(n, width, device="cuda")  # noqa: E731
    dy, dx, w1, w2 = new(), new(), torch.zeros(width, device="cuda"), torch.zeros(width, device="cuda")
    ws = torch.zeros(L.workspace_bytes(n), dtype=torch.uint8, device="cuda")
    L.backward([y.cuda()], [dh.cuda()], [dy], n, residual_out=r.cuda(), grad_residual=dx, grad_post_weight=w1, grad_pre_weight=w2, workspace=ws)
    torch.cuda.synchronize()
    p = dict(p, post_eps=float(torch.tensor(1e-37)), pre_eps=float(torch.tensor(1e-37)))
    want = ref.backward(y.double()[None], r.double(), dh.double()[None], torch.zeros(n, width, dtype=torch.float64), None, 0, p)
    within(dx[:3], tuple(v[:3] for v in want["grad_residual"]), "f32", "dx")
    assert bool((dx[2] == 0).all()) and bool(torch.isfinite(dx).all())
    keep = [0, 2, 4]  # (the row of zeros in y: its gradient is past 10^18 times the others')
    within(dy[keep], tuple(v[keep] for v in want["grad_ins"]), "f32", "dy")
    assert not bool(torch.isnan(dy).any()) and not bool(torch.isnan(w1).any()) and not bool(torch.isnan(w2).any())


def test_no_rows(hip):
    """Gradients of parameters over no rows are zero; nothing of rows or gate is touched."""
    import torch
    for width in (3, 700, 9000):
        gen = torch.Generator().manual_seed(6)
        p = params(torch, gen, width, "f32", "layer", "layer", biases=True)
        L = layer_of(hip, "f32", width, p)
        w = [torch.full((width,), 7.0, device="cuda") for _ in range(4)]
        ws = torch.full((L.workspace_bytes(0, 3),), 0x5A, dtype=torch.uint8, device="cuda")
        L.backward([None], [None], [None], 0, gate=0x1000, gate_rows=3, grad_gate=0x2000, grad_post_weight=w[0], grad_post_bias=w[1], grad_pre_weight=w[2],
                   grad_pre_bias=w[3], workspace=ws)
        L.forward([None], [None], 0, gate=0x1000, gate_rows=3)
        torch.cuda.synchronize()
        assert all(bool((v == 0).all()) for v in w)


@pytest.mark.parametrize("n,width,gate_rows,biases", [(300, 8192, 1, False), (300, 8192, 1, True), (300, 8200, 1, False), (290, 9000, 1, True), (4500, 40, 1, True),
                                                      (2100, 600, 1, False), (101, 600, 100, True), (5000, 64, 2, True), (700, 4100, 2, True)])
def test_more_gate_rows_than_teams(hip, n, width, gate_rows, biases):
    """A team then goes through several gate rows and keeps its sums over them; and a last gate row of one row."""
    import torch
    gen = torch.Generator().manual_seed(14)
    p = params(torch, gen, width, "bf16", "rms", "layer", biases=biases)
    L = layer_of(hip, "bf16", width, p)
    groups = -(-n // gate_rows)
    y, r, dh, dr = (rows(torch, gen, "bf16", n, width) for _ in range(4))
    gate = rows(torch, gen, "bf16", groups, width)
    want = ref.backward(y.double()[None], r.double(), dh.double()[None], dr.double(), gate.double(), gate_rows, p)
    dy, dx, dg = torch.zeros_like(y, device="cuda"), torch.zeros_like(y, device="cuda"), torch.zeros_like(gate, device="cuda")
    names = ["post_weight", "pre_weight"] + (["post_bias", "pre_bias"] if biases else [])
    w = {k: torch.zeros(width, dtype=torch.bfloat16, device="cuda") for k in names}
    ws = torch.full((L.workspace_bytes(n, gate_rows),), 0x5A, dtype=torch.uint8, device="cuda")
    L.backward([y.cuda()], [dh.cuda()], [dy], n, residual_out=r.cuda(), grad_residual_out=dr.cuda(), grad_residual=dx, gate=gate.cuda(), gate_rows=gate_rows,
               grad_gate=dg, workspace=ws, **{"grad_" + k: v for k, v in w.items()})
    torch.cuda.synchronize()
    within(dx, want["grad_residual"], "bf16", "dx")
    within(dy, want["grad_ins"], "bf16", "dy")
    within(dg, want["grad_gate"], "bf16", "gate")
    for k in names:
        within(w[k], want["grad_" + k], "bf16", k)


@pytest.mark.parametrize("dtype,width,n_in,n_out", [("bf16", 4096, 4, 3), ("f32", 8192, 3, 2), ("f16", 12000, 8, 1), ("f32", 10000, 3, 1), ("bf16", 400, 5, 2)])
def test_large_calls_give_the_bits_of_small_ones(hip, dtype, width, n_in, n_out):
    """Beyond the Infinity Cache rows are read non-temporally, by instances of their own: the same rows in slices of less."""
    import torch
    size = 4 if dtype == "f32" else 2
    n = (300 << 20) // (width * size * (n_in + n_out + 2)) + 7
    gen = torch.Generator().manual_seed(15)
    p = params(torch, gen, width, dtype, "layer", "rms", biases=True)
    L = layer_of(hip, dtype, width, p)
    t = ref.TYPES[dtype]
    dev = torch.Generator(device="cuda").manual_seed(15)
    make = lambda: torch.randn(n, width, device="cuda", generator=dev).to(t)  # noqa: E731
    parts, x = [make() for _ in range(n_in)], make()
    got = [torch.zeros_like(x) for _ in range(2 + n_out)]
    want = [torch.zeros_like(x) for _ in range(2 + n_out)]
    L.forward(parts, got[2:], n, residual=x, residual_out=got[0], folded=got[1])
    step = n // 5 + 1
    for lo in range(0, n, step):
        cut = lambda v: v[lo:lo + step]  # noqa: E731
        L.forward([cut(v) for v in parts], [cut(v) for v in want[2:]], cut(x).shape[0], residual=cut(x), residual_out=cut(want[0]), folded=cut(want[1]))
    torch.cuda.synchronize()
    for a, b in zip(got, want):
        assert torch.equal(a, b)
    # the backward pass reads four rows and writes two for each
    n = min(n, (300 << 20) // (width * size * 6) + 7) if n * width * size * 5 > (300 << 20) else n
    y, r, dh, dr = (v[:n] for v in (parts + [x, got[0], got[1]])[:4])
    a, b = [torch.zeros_like(y) for _ in range(2)], [torch.zeros_like(y) for _ in range(2)]
    L.backward([y], [dh], [a[0]], n, residual_out=r, grad_residual_out=dr, grad_residual=a[1])
    step = n // 5 + 1
    for lo in range(0, n, step):
        cut = lambda v: v[lo:lo + step]  # noqa: E731
        L.backward([cut(y)], [cut(dh)], [cut(b[0])], cut(y).shape[0], residual_out=cut(r), grad_residual_out=cut(dr), grad_residual=cut(b[1]))
    torch.cuda.synchronize()
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


@pytest.mark.parametrize("fmt,dtype,heads,dim", [("f8e4m3", "bf16", 8, 128), ("f4e2m1", "f16", 1, 64), ("i8", "f32", 3, 80), ("f8e5m2", "bf16", 7, 61), ("f4e2m1", "bf16", 2, 33),
                                                 ("i8", "f16", 9, 72), ("f8e4m3", "f32", 1, 20)])
def test_large_cache_calls_give_the_bits_of_small_ones(hip, fmt, dtype, heads, dim):
    """Large calls keep several tokens of a wavefront in flight and read their sources non-temporally, by instances of their own."""
    import torch
    t = ref.TYPES[dtype]
    n = (100 << 20) // (heads * dim * (4 if dtype == "f32" else 2)) + 13
    page = 48
    pages = -(-n // page) + 1
    row, blocks = hip.Cache.row_bytes(fmt, dim)
    dev = torch.Generator(device="cuda").manual_seed(16)
    x = (torch.randn(n, heads, dim, device="cuda", generator=dev) * torch.exp(2 * torch.randn(n, heads, 1, device="cuda", generator=dev))).to(t)
    slots = torch.randperm(pages * page, device="cuda", generator=dev)[:n].clone()
    slots[torch.rand(n, device="cuda", generator=dev) < 0.02] = -1
    held = []
    for step in (n, n // 400 + 1):
        codes, scales = torch.zeros(pages, page, heads, row, dtype=torch.uint8, device="cuda"), torch.zeros(pages, page, heads, blocks, dtype=torch.uint8, device="cuda")
        c = hip.Cache(fmt, heads, dim, page, pages, [codes], [scales])
        for lo in range(0, n, step):
            part = x[lo:lo + step]
            c.write(dtype, [part], slots[lo:lo + step], part.shape[0])
        held.append((codes, scales, c))
    torch.cuda.synchronize()
    assert torch.equal(held[0][0], held[1][0]) and torch.equal(held[0][1], held[1][1])
    c = held[0][2]
    table = torch.randperm(pages, device="cuda", generator=dev).int()
    out, want = torch.full((pages * page, heads, dim), 3.0, dtype=t, device="cuda"), torch.full((pages * page, heads, dim), 3.0, dtype=t, device="cuda")
    most = pages * page - 5
    c.read(dtype, [out], table[None], torch.tensor([most], dtype=torch.int32, device="cuda"), 1, pages * page)
    some = pages // 300 + 1
    for lo in range(0, pages, some):
        part = table[lo:lo + some].contiguous()
        length = min(part.numel() * page, most - lo * page)
        c.read(dtype, [want[lo * page:]], part[None], torch.tensor([length], dtype=torch.int32, device="cuda"), 1, part.numel() * page)
    torch.cuda.synchronize()
    assert torch.equal(out.view(torch.uint8), want.view(torch.uint8))


def test_captured_and_replayed(hip):
    """Forward, backward, cache write and read recorded into a graph and replayed five times on new inputs, with eager calls and
    synchronizations between: every replay gives the bits of the eager call."""
    import torch
    gen = torch.Generator().manual_seed(8)
    n, width, heads, dim, page = 50, 1500, 4, 64, 16
    p = params(torch, gen, width, "bf16", "layer", "rms", biases=True)
    L = layer_of(hip, "bf16", width, p)
    gate = rows(torch, gen, "bf16", 5, width).cuda()
    make = lambda: [rows(torch, gen, "bf16", n, width).cuda() for _ in range(5)]  # noqa: E731
    y, x, dh, dr, kv = make()
    pages = 8
    row, blocks = hip.Cache.row_bytes("f4e2m1", dim)
    slots = torch.randperm(pages * page, generator=gen)[:n].cuda()
    table, lengths = torch.randperm(pages, generator=gen).int().view(2, 4).cuda(), torch.tensor([50, 33], dtype=torch.int32).cuda()

    def buffers():
        b = {k: torch.zeros_like(y) for k in ("r", "h", "dy", "dx")} | {"dg": torch.zeros_like(gate)}
        b |= {"d" + k: torch.zeros(width, dtype=torch.bfloat16, device="cuda") for k in ("post_weight", "post_bias", "pre_weight", "pre_bias")}
        b["codes"], b["scales"] = torch.zeros(pages, page, heads, row, dtype=torch.uint8, device="cuda"), torch.zeros(pages, page, heads, blocks, dtype=torch.uint8, device="cuda")
        b["out"] = torch.zeros(2, 64, heads, dim, dtype=torch.bfloat16, device="cuda")
        b["ws"] = torch.zeros(L.workspace_bytes(n, 11), dtype=torch.uint8, device="cuda")
        return b

    def step(b):
        s = torch.cuda.current_stream().cuda_stream
        L.forward([y], [b["h"]], n, residual=x, residual_out=b["r"], gate=gate, gate_rows=11, stream=s)
        L.backward([y], [dh], [b["dy"]], n, residual_out=b["r"], grad_residual_out=dr, grad_residual=b["dx"], gate=gate, gate_rows=11, grad_gate=b["dg"],
                   grad_post_weight=b["dpost_weight"], grad_post_bias=b["dpost_bias"], grad_pre_weight=b["dpre_weight"], grad_pre_bias=b["dpre_bias"],
                   workspace=b["ws"], stream=s)
        c = hip.Cache("f4e2m1", heads, dim, page, pages, [b["codes"]], [b["scales"]])
        c.write("bf16", [b["h"]], slots, n, stream=s, token_stride=width, head_stride=dim)
        c.read("bf16", [b["out"]], table, lengths, 2, 64, stream=s)

    eager, held = buffers(), buffers()
    step(held)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        step(held)
    for k in range(5):
        for v in (y, x, dh, dr, gate):
            v.copy_(rows(torch, gen, "bf16", *v.shape))
        step(eager)
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        for name in eager:
            if name != "ws":
                assert torch.equal(eager[name].view(torch.uint8), held[name].view(torch.uint8)), "replay %d: %s" % (k, name)


def test_other_streams_and_threads(hip):
    """The same layer object and cache from two threads on two streams at once, each with its own buffers."""
    import torch
    gen = torch.Generator().manual_seed(9)
    n, width = 300, 2048
    p = params(torch, gen, width, "bf16")
    L = layer_of(hip, "bf16", width, p)
    codes, scales = torch.zeros(2, 64, 16, 8, 128, dtype=torch.uint8, device="cuda"), torch.zeros(2, 64, 16, 8, 4, dtype=torch.uint8, device="cuda")
    cache = hip.Cache("f8e4m3", 8, 128, 16, 64, [codes[0]], [scales[0]])
    sets, wrong = [], []
    for k in range(2):
        y, dh = rows(torch, gen, "bf16", n, width), rows(torch, gen, "bf16", n, width)
        sets.append(dict(y=y.cuda(), dh=dh.cuda(), kv=rows(torch, gen, "bf16", n, 8, 128), h=torch.zeros(n, width, dtype=torch.bfloat16, device="cuda"),
                         dy=torch.zeros(n, width, dtype=torch.bfloat16, device="cuda"), w=torch.zeros(2, width, dtype=torch.bfloat16, device="cuda"),
                         ws=torch.zeros(L.workspace_bytes(n), dtype=torch.uint8, device="cuda"), slots=(torch.arange(n) + 400 * k).cuda(),
                         fwd=ref.forward(y.double()[None], None, None, 0, p), cpu=(y, dh)))
    for s in sets:
        s["d_kv"] = s["kv"].cuda()
    torch.cuda.synchronize()

    def work(s):
        try:
            stream = torch.cuda.Stream()
            for _ in range(20):
                L.forward([s["y"]], [s["h"]], n, stream=stream.cuda_stream)
                L.backward([s["y"]], [s["dh"]], [s["dy"]], n, residual_out=s["y"], grad_post_weight=s["w"][0], grad_pre_weight=s["w"][1], workspace=s["ws"],
                           stream=stream.cuda_stream)
                cache.write("bf16", [s["d_kv"]], s["slots"], n, stream=stream.cuda_stream)
            stream.synchronize()
        except Exception as e:  # noqa: BLE001
            wrong.append(e)

    threads = [threading.Thread(target=work, args=(s,)) for s in sets]
    [t.start() for t in threads]
    [t.join() for t in threads]
    torch.cuda.synchronize()
    assert not wrong, wrong
    for k, s in enumerate(sets):
        within(s["h"], s["fwd"]["outs"], "bf16", "thread %d" % k)
        y, dh = s["cpu"]
        want = ref.backward(y.double()[None], y.double(), dh.double()[None], torch.zeros(n, width, dtype=torch.float64), None, 0, p)
        within(s["dy"], want["grad_ins"], "bf16", "thread %d, dy" % k)
        within(s["w"][0], want["grad_post_weight"], "bf16", "thread %d, weights" % k)
        got, _ = cref.encode("f8e4m3", s["kv"].double())
        assert torch.equal(codes[0].view(-1, 8, 128)[s["slots"]].cpu(), got)


def test_cache_offsets_beyond_32_bits(hip):
    """Pages, rows of the source and rows of the output past 4 GiB from the first."""
    import torch
    heads, dim, page = 2, 64, 4
    gen = torch.Generator().manual_seed(10)
    page_stride = (3 << 30) + 128  # pages 0, 1 and 2 at 0, 3 and 6 GiB
    big = torch.empty(2 * page_stride + 4096, dtype=torch.uint8, device="cuda")
    scales = torch.zeros(3, page, heads, 2, dtype=torch.uint8, device="cuda")
    c = hip.Cache("i8", heads, dim, page, 3, [big], [scales], code_strides=(page_stride, heads * dim, dim))
    x = rows(torch, gen, "f16", 3, heads, dim)
    far = (1 << 31) - 64  # elements from one token of the source to the next: 4 GiB less a little
    src = torch.empty(2 * far + heads * dim, dtype=torch.float16, device="cuda")
    for t in range(3):
        src[t * far:t * far + heads * dim] = x[t].reshape(-1).cuda()
    slots = torch.tensor([9, 2, 5], device="cuda")  # pages 2, 0, 1
    c.write("f16", [src], slots, 3, token_stride=far)
    table = torch.tensor([[0, 1, 2]], dtype=torch.int32, device="cuda")
    src.zero_()
    c.read("f16", [src], torch.tensor([[2]], dtype=torch.int32, device="cuda"), torch.tensor([2], dtype=torch.int32, device="cuda"), 1, 2, token_stride=far)
    torch.cuda.synchronize()
    codes, sc = cref.encode("i8", x.double())
    back = cref.decode("i8", codes, sc, dim, "f16")
    assert cref.same(src[far:far + heads * dim].view(heads, dim), back[0])   # slot 9 = page 2, its token 1
    out = torch.zeros(12, heads, dim, dtype=torch.float16, device="cuda")
    c.read("f16", [out], table, torch.tensor([12], dtype=torch.int32, device="cuda"), 1, 12)
    torch.cuda.synchronize()
    for i, slot in enumerate((9, 2, 5)):
        assert cref.same(out[slot], back[i])


def test_cache_lengths_that_promise_too_much(hip):
    """Lengths below 0 and beyond max_len and the table, rows beyond the output, pages that are not there: nothing is read or written
    for them."""
    import torch
    heads, dim, page, pages = 1, 32, 4, 5
    gen = torch.Generator().manual_seed(11)
    codes = torch.randint(-127, 128, (pages, page, heads, dim), generator=gen, dtype=torch.int8).view(torch.uint8)
    scales = torch.full((pages, page, heads, 1), 127, dtype=torch.uint8)
    c = hip.Cache("i8", heads, dim, page, pages, [codes.cuda()], [scales.cuda()])
    table = torch.tensor([[0, 1], [2, 3], [4, -1], [7, 2], [1, 1]], dtype=torch.int32).cuda()
    lengths = torch.tensor([-3, 1000, 8, 8, 8], dtype=torch.int32).cuda()
    start = torch.tensor([0, 0, 9, 20, 1 << 40], dtype=torch.int64).cuda()
    out = torch.full((26, heads, dim), 9.0, device="cuda")
    c.read("f32", [out], table, lengths, 5, 9, row_start=start, out_rows=26)
    torch.cuda.synchronize()
    want = torch.full((26, heads, dim), 9.0)
    v = cref.decode("i8", codes, scales, dim, "f32")
    want[0:8] = v[[2, 3]].flatten(0, 1)      # 1000 tokens: max_len 9, the table's two pages
    want[9:13] = v[4]                        # the second page is not there
    want[24:26] = v[2][:2]                   # the first is not, the last rows are beyond the output
    assert cref.same(out, want)


@pytest.mark.parametrize("fmt", ["f8e4m3", "f4e2m1"])
def test_a_layers_step_over_resident_ranks(hip, oracle, fmt):
    """Eight ranks' partial outputs -> norms, stored to every rank -> each rank projects keys and values -> its cache -> pages moved to
    another cache by one graph of copies -> read there; every stage against 64 bits from the stage before."""
    import torch
    gen = torch.Generator().manual_seed(12)
    world, n, width, heads, dim, page = 8, 45, 512, 2, 64, 16
    p = params(torch, gen, width, "bf16")
    L = layer_of(hip, "bf16", width, p)
    parts, x = rows(torch, gen, "bf16", world, n, width, scale=0.4), rows(torch, gen, "bf16", n, width)
    d_parts, d_x = parts.cuda(), x.cuda()
    h, stream = torch.zeros(world, n, width, dtype=torch.bfloat16, device="cuda"), torch.cuda.current_stream().cuda_stream
    L.forward(list(d_parts), list(h), n, residual=d_x, residual_out=d_x, stream=stream)
    torch.cuda.synchronize()
    want = ref.forward(parts.double(), x.double(), None, 0, p)
    within(d_x, want["residual_out"], "bf16", "r")
    for r in range(world):
        within(h[r], want["outs"], "bf16", "h of rank %d" % r)
    pages, row, blocks = 4, *hip.Cache.row_bytes(fmt, dim)
    size, ssize = page * heads * row, page * heads * blocks
    new = lambda b: torch.zeros(world, 2, pages, page, heads, b, dtype=torch.uint8, device="cuda")  # noqa: E731
    codes, scales, codes2, scales2 = new(row), new(blocks), new(row), new(blocks)
    slots = torch.arange(n).cuda()
    kv = torch.zeros(world, 2, n, heads, dim, dtype=torch.bfloat16, device="cuda")
    for r in range(world):
        w = rows(torch, gen, "bf16", 2, width, heads * dim, scale=width ** -0.5).cuda()
        for k in range(2):
            kv[r, k] = (h[r].float() @ w[k].float()).to(torch.bfloat16).view(n, heads, dim)
        hip.Cache(fmt, heads, dim, page, pages, list(codes[r]), list(scales[r])).write("bf16", list(kv[r]), slots, n, stream=stream)
    moved = [3, 0, 2, 1]  # page k of a rank goes to page moved[k] of the other cache
    ops = []
    for r in range(world):
        for k in range(2):
            for a in range(3):
                ops.append(dict(dtype="f8e4m3", ins=[codes[r, k, a]], outs=[codes2[r, k, moved[a]]], count=size))
                ops.append(dict(dtype="f8e4m3", ins=[scales[r, k, a]], outs=[scales2[r, k, moved[a]]], count=ssize))
    g = hip.Graph(ops)
    g.run(stream)
    assert g.status(stream) == (len(ops), len(ops))
    table, lengths = torch.tensor([moved[:3]], dtype=torch.int32).cuda(), torch.tensor([n], dtype=torch.int32).cuda()
    for r in range(world):
        out = torch.zeros(2, n, heads, dim, dtype=torch.bfloat16, device="cuda")
        hip.Cache(fmt, heads, dim, page, pages, list(codes2[r]), list(scales2[r])).read("bf16", list(out), table, lengths, 1, n, stream=stream)
        torch.cuda.synchronize()
        for k in range(2):
            c, s = cref.encode(fmt, kv[r, k].cpu().double())
            assert cref.same(out[k], cref.decode(fmt, c, s, dim, "bf16")), "rank %d tensor %d" % (r, k)
    g.destroy()


def test_two_blocks_trained_over_resident_ranks(hip, oracle):
    """Two layers one behind the other, forward and backward, two ranks' partial outputs and partial gradients: the gradients of a
    chain against automatic differentiation of the same chain in 64 bits.  Bounds are of one layer, so the
    comparison is by 2-norm: each stored tensor is off by at most 2^-24 of itself per operation (f32), some 200 operations deep."""
    import torch
    gen = torch.Generator().manual_seed(13)
    n, width = 24, 320
    ps = [params(torch, gen, width, "f32", "rms", "layer", biases=True), params(torch, gen, width, "f32", "layer", "rms", biases=True)]
    mix = [torch.randn(2, width, width, generator=gen) * width ** -0.5 for _ in range(2)]   # what a block does to h on either rank
    x, seed_h, seed_r = (torch.randn(n, width, generator=gen) for _ in range(3))
    block0 = torch.randn(2, n, width, generator=gen)
    Ls = [layer_of(hip, "f32", width, p) for p in ps]
    new = lambda *s: torch.zeros(*s, device="cuda")  # noqa: E731
    # forward: layer 0 takes block0's parts and x; layer 1 the parts mixed from h0 and r0
    parts = [block0.cuda(), new(2, n, width)]
    r, h, y, d_mix = [new(n, width) for _ in range(2)], [new(2, n, width) for _ in range(2)], [new(n, width) for _ in range(2)], [m.cuda() for m in mix]
    Ls[0].forward(list(parts[0]), list(h[0]), n, residual=x.cuda(), residual_out=r[0], folded=y[0])
    for k in range(2):
        parts[1][k] = (h[0][k].double() @ d_mix[0][k].double()).float()
    Ls[1].forward(list(parts[1]), list(h[1]), n, residual=r[0], residual_out=r[1], folded=y[1])
    # backward
    names = ("post_weight", "post_bias", "pre_weight", "pre_bias")
    grads = [{k: new(width) for k in names} for _ in range(2)]
    ws = new(Ls[0].workspace_bytes(n) // 4 + 1)
    dy, dx = [new(2, n, width) for _ in range(2)], [new(n, width) for _ in range(2)]
    dh1 = torch.stack([seed_h * 0.25, seed_h * 0.75]).cuda()
    Ls[1].backward([y[1]], list(dh1), list(dy[1]), n, residual_out=r[1], grad_residual_out=seed_r.cuda(), grad_residual=dx[1], workspace=ws,
                   **{"grad_" + k: grads[1][k] for k in names})
    dh0 = torch.stack([(dy[1][k].double() @ d_mix[0][k].double().T).float() for k in range(2)])
    Ls[0].backward([y[0]], list(dh0), list(dy[0]), n, residual_out=r[0], grad_residual_out=dx[1], grad_residual=dx[0], workspace=ws,
                   **{"grad_" + k: grads[0][k] for k in names})
    torch.cuda.synchronize()
    leaves = {(k, name): ps[k][name].clone().requires_grad_() for k in range(2) for name in names}
    b64, x64 = block0.double().requires_grad_(), x.double().requires_grad_()
    f0 = ref.forward(b64, x64, None, 0, dict(ps[0], **{m: leaves[0, m] for m in names}))
    parts1 = torch.stack([f0["outs"][0] @ mix[0][k].double() for k in range(2)])
    f1 = ref.forward(parts1, f0["residual_out"][0], None, 0, dict(ps[1], **{m: leaves[1, m] for m in names}))
    ((f1["outs"][0] * seed_h.double()).sum() + (f1["residual_out"][0] * seed_r.double()).sum()).backward()
    pairs = [(dy[0][0], b64.grad[0], "dy"), (dy[0][1], b64.grad[1], "dy of the second rank"), (dx[0], x64.grad, "dx")]
    pairs += [(grads[k][m], leaves[k, m].grad, "%s of layer %d" % (m, k)) for k in range(2) for m in names]
    for got, want, what in pairs:
        off = float((got.double().cpu() - want).norm() / want.norm())
        assert off <= 200 * 2.0 ** -24 * 8, "%s off by %.3g" % (what, off)
