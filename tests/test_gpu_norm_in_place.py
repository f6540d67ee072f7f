"""The norms written over their own inputs in every form that goes about its rows in its own way: with the next row on its way and without, of
one or several gradients and partial outputs, in strips of a gate row, in every type; and operands on their way out of scope."""
import pytest

import norm_reference as ref
import test_gpu_norm_cache_use as use

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("gate_rows", [0, 1, 3, 400])
@pytest.mark.parametrize("n_in,n_out", [(1, 1), (1, 3), (2, 2), (3, 1)])
@pytest.mark.parametrize("dtype,width", [("f32", 40), ("f32", 300), ("f32", 1025), ("f32", 4100), ("f32", 8200), ("bf16", 72), ("bf16", 520), ("bf16", 4097),
                                         ("bf16", 8301), ("f16", 333), ("f16", 2048), ("f16", 9001)])
def test_backward_in_place(hip, dtype, width, n_in, n_out, gate_rows):
    """dy over every partial output and every gradient of h, dx over the gradient from further on or over r."""
    import torch
    gen = torch.Generator().manual_seed(width + 7 * n_in + n_out + gate_rows)
    n = 600 if width < 1000 else 290  # (several rows a team)
    if width < 100:
        n = 4500
    kinds = [("rms", "rms"), ("layer", "rms"), ("rms", "layer"), ("layer", "layer")][(width + n_in + gate_rows) % 4]
    p = use.params(torch, gen, width, dtype, *kinds, biases=n_out != 2)
    L = use.layer_of(hip, dtype, width, p)
    y, dh = use.rows(torch, gen, dtype, n_in, n, width, scale=0.7), use.rows(torch, gen, dtype, n_out, n, width)
    r, dr = use.rows(torch, gen, dtype, n, width), use.rows(torch, gen, dtype, n, width)
    gate = use.rows(torch, gen, dtype, -(-n // gate_rows), width) if gate_rows else None
    want = ref.backward(y.double(), r.double(), dh.double().clone(), dr.double(), None if gate is None else gate.double(), gate_rows, p)
    d_gate = None if gate is None else gate.cuda()
    ws = torch.zeros(L.workspace_bytes(n, gate_rows), dtype=torch.uint8, device="cuda")
    for over_r in (False, True):
        d_y, d_dh, d_r, d_dr = list(y.cuda()), list(dh.cuda()), r.cuda(), dr.cuda()
        dx = d_r if over_r else d_dr
        dg = None if gate is None else torch.zeros_like(d_gate)
        w = {k: torch.zeros(width, dtype=ref.TYPES[dtype], device="cuda") for k in ("post_weight", "post_bias", "pre_weight", "pre_bias") if p[k] is not None}
        L.backward(d_y, d_dh, d_y + d_dh, n, residual_out=d_r, grad_residual_out=d_dr, grad_residual=dx, gate=d_gate, gate_rows=gate_rows, grad_gate=dg,
                   workspace=ws, **{"grad_" + k: v for k, v in w.items()})
        torch.cuda.synchronize()
        for k, b in enumerate(d_y + d_dh):
            use.within(b, want["grad_ins"], dtype, "grad_ins %d" % k)
        use.within(dx, want["grad_residual"], dtype, "grad_residual")
        if gate is not None:
            use.within(dg, want["grad_gate"], dtype, "grad_gate")
        for k, b in w.items():
            use.within(b, want["grad_" + k], dtype, k)


@pytest.mark.parametrize("gate_rows", [0, 2])
@pytest.mark.parametrize("dtype,width", [("f32", 24), ("f32", 4000), ("f32", 9000), ("bf16", 513), ("bf16", 16384), ("f16", 7), ("f16", 1025), ("f16", 8193)])
def test_forward_in_place(hip, dtype, width, gate_rows):
    """y over the first of three partial outputs, h over the others and a copy, r over x."""
    import torch
    gen = torch.Generator().manual_seed(width + gate_rows)
    n = 61
    p = use.params(torch, gen, width, dtype, "layer", "rms", biases=True)
    parts, x = use.rows(torch, gen, dtype, 3, n, width), use.rows(torch, gen, dtype, n, width)
    gate = use.rows(torch, gen, dtype, -(-n // gate_rows), width) if gate_rows else None
    want = ref.forward(parts.double(), x.double(), None if gate is None else gate.double(), gate_rows, p)
    d, d_x, copy = list(parts.cuda()), x.cuda(), torch.zeros(n, width, dtype=x.dtype, device="cuda")
    use.layer_of(hip, dtype, width, p).forward(d, [d[1], copy, d[2]], n, residual=d_x, residual_out=d_x, folded=d[0],
                                               gate=None if gate is None else gate.cuda(), gate_rows=gate_rows)
    torch.cuda.synchronize()
    use.within(d[0], want["folded"], dtype, "folded")
    use.within(d_x, want["residual_out"], dtype, "residual_out")
    for b in (d[1], d[2], copy):
        use.within(b, want["outs"], dtype, "outs")


def test_workspace_let_go_behind_the_call(hip):
    """A workspace recorded on the call's stream may go out of scope right behind the call, whatever the allocator's own stream does next."""
    import torch
    gen = torch.Generator().manual_seed(1)
    n, width = 6000, 4096
    p = use.params(torch, gen, width, "bf16", biases=True)
    L = use.layer_of(hip, "bf16", width, p)
    y, r, dh = (use.rows(torch, gen, "bf16", n, width).cuda() for _ in range(3))
    names = ("post_weight", "post_bias", "pre_weight", "pre_bias")
    need, stream = L.workspace_bytes(n), torch.cuda.Stream()
    found = []
    for k in range(4):
        dy, w = torch.zeros_like(y), {"grad_" + m: torch.zeros(width, dtype=torch.bfloat16, device="cuda") for m in names}
        torch.cuda.synchronize()
        workspace = torch.empty(need, dtype=torch.uint8, device="cuda")
        stream.wait_stream(torch.cuda.current_stream())
        L.backward([y], [dh], [dy], n, residual_out=r, workspace=workspace, stream=stream.cuda_stream, **w)
        if k:
            workspace.record_stream(stream)
            del workspace
            for _ in range(3):  # (on the current stream: what another part of a program does with memory that is free again)
                torch.full((need,), 0x7F, dtype=torch.uint8, device="cuda")
        torch.cuda.synchronize()
        found.append([dy] + list(w.values()))
    for later in found[1:]:
        assert all(torch.equal(a, b) for a, b in zip(found[0], later))


def test_pinned_host_memory_passes(hip):
    """What the GPU can reach is taken: slots, table and lengths that the host writes in pinned memory, and weights."""
    import torch
    gen = torch.Generator().manual_seed(2)
    heads, dim, page, pages, n = 2, 64, 4, 6, 20
    codes, scales = (torch.zeros(pages, page, heads, k, dtype=torch.uint8, device="cuda") for k in (dim, 2))
    cache = hip.Cache("i8", heads, dim, page, pages, [codes], [scales])
    x = use.rows(torch, gen, "bf16", n, heads, dim)
    pinned = lambda v: torch.empty(v.shape, dtype=v.dtype, pin_memory=True).copy_(v)  # noqa: E731
    slots, table, lengths = pinned(torch.arange(n)), pinned(torch.arange(pages, dtype=torch.int32)[None]), pinned(torch.tensor([n], dtype=torch.int32))
    out = torch.zeros(n, heads, dim, dtype=torch.bfloat16, device="cuda")
    cache.write("bf16", [x.cuda()], slots, n)
    cache.read("bf16", [out], table, lengths, 1, n)
    torch.cuda.synchronize()
    assert use.cref.same(out, use.cref.decode("i8", *use.cref.encode("i8", x.double()), dim, "bf16"))
    w = pinned(torch.full((64,), 2.0))
    a, b = torch.zeros(2, 64, device="cuda"), torch.zeros(2, 64, device="cuda")
    rows = torch.randn(2, 64, generator=gen).cuda()
    hip.FoldNorm("f32", 64, pre_weight=w).forward([rows], [a], 2)
    hip.FoldNorm("f32", 64, pre_weight=w.cuda()).forward([rows], [b], 2)
    torch.cuda.synchronize()
    assert torch.equal(a, b)
    with pytest.raises(hip.PcclError):
        hip.FoldNorm("f32", 64, pre_weight=torch.ones(64))
