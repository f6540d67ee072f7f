"""The norms and the cache on the default streams by each of their handles."""
import pytest

import cache_reference as cref
import norm_reference as ref
import test_gpu_norm_cache_use as use

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("stream", [None, 0, 1, 2], ids=["none", "null", "legacy", "per-thread"])
def test_default_stream(hip, stream):
    import torch
    gen = torch.Generator().manual_seed(1)
    n, width, heads, dim = 9, 512, 2, 64
    p = use.params(torch, gen, width, "bf16")
    L = use.layer_of(hip, "bf16", width, p)
    y, r, dh, kv = (use.rows(torch, gen, "bf16", n, width) for _ in range(4))
    d_y, d_r, d_dh, d_kv = y.cuda(), r.cuda(), dh.cuda(), kv.cuda()
    h, dy, out = torch.zeros_like(d_y), torch.zeros_like(d_y), torch.zeros(n, heads, dim, dtype=torch.bfloat16, device="cuda")
    w, ws = torch.zeros(width, dtype=torch.bfloat16, device="cuda"), torch.zeros(L.workspace_bytes(n), dtype=torch.uint8, device="cuda")
    cache = hip.Cache("i8", heads, dim, 4, 3, [torch.zeros(3 * 4 * heads * dim, dtype=torch.uint8, device="cuda")],
                      [torch.zeros(3 * 4 * heads * 2, dtype=torch.uint8, device="cuda")])
    slots, table, lengths = torch.arange(n).cuda(), torch.arange(3, dtype=torch.int32)[None].cuda(), torch.tensor([n], dtype=torch.int32).cuda()
    torch.cuda.synchronize()
    L.forward([d_y], [h], n, stream=stream)
    L.backward([d_y], [d_dh], [dy], n, residual_out=d_r, grad_pre_weight=w, workspace=ws, stream=stream)
    cache.write("bf16", [d_kv], slots, n, stream=stream, token_stride=width)
    cache.read("bf16", [out], table, lengths, 1, n, stream=stream)
    torch.cuda.synchronize()
    use.within(h, ref.forward(y.double()[None], None, None, 0, p)["outs"], "bf16", "h")
    want = ref.backward(y.double()[None], r.double(), dh.double()[None], torch.zeros(n, width, dtype=torch.float64), None, 0, p)
    use.within(dy, want["grad_ins"], "bf16", "dy")
    use.within(w, want["grad_pre_weight"], "bf16", "weight")
    kv = kv[:, :heads * dim].reshape(n, heads, dim)
    assert cref.same(out, cref.decode("i8", *cref.encode("i8", kv.double()), dim, "bf16"))
