"""Elements at, right below and right above every tie between two codes, under small, ordinary and large scales: a binary32 has 20 bits
below an element's last one, and all of them decide."""
import pytest

import cache_reference as ref

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("fmt", ["f8e4m3", "f8e5m2", "i8", "f4e2m1"])
def test_write_next_to_ties(hip, fmt, dtype):
    import torch
    t = ref.TYPES[dtype]
    g = torch.tensor(ref.grid(fmt), dtype=torch.float64)
    near = torch.cat([(g[1:] + g[:-1]) / 2, g]).to(t)  # (exact: one bit more than a code has)
    near = torch.cat([near, torch.nextafter(near, torch.tensor(float("inf"), dtype=t)), torch.nextafter(near, torch.tensor(-float("inf"), dtype=t))])
    near = torch.cat([near, -near])
    near = near[near.double().abs() <= g[-1]]
    near = torch.cat([near, near[:-near.numel() % 31]]).view(-1, 31).double()
    lead = g[-1].expand(near.shape[0], 1)  # every block has the format's largest value in it, so that its scale is that power of two
    spread = range(-149, 114) if dtype != "f16" else range(-24, 1)
    x = torch.cat([(torch.cat([lead, near], 1) * 2.0 ** k).to(t) for k in spread if float(g[-1]) * 2.0 ** k <= torch.finfo(t).max])[:, None].contiguous()
    n = x.shape[0]
    codes, scales = ref.encode(fmt, x.double())
    row = codes.shape[-1]
    dev_codes, dev_scales = torch.zeros(n, 1, 1, row, dtype=torch.uint8, device="cuda"), torch.zeros(n, 1, 1, 1, dtype=torch.uint8, device="cuda")
    hip.Cache(fmt, 1, 32, 1, n, [dev_codes], [dev_scales]).write(dtype, [x.cuda()], torch.arange(n, device="cuda"), n)
    torch.cuda.synchronize()
    assert torch.equal(dev_scales.cpu().view(n, 1, 1), scales)
    off = (dev_codes.cpu().view(n, row) != codes.view(n, row)).any(-1)
    assert not bool(off.any()), "%d of %d blocks, first %s" % (int(off.sum()), n, x[off][0])


@pytest.mark.parametrize("fmt", ["f8e4m3", "f8e5m2", "i8", "f4e2m1"])
def test_write_any_binary32(hip, fmt):
    """Bits at random, the exponents of a block near each other."""
    import torch
    gen = torch.Generator().manual_seed(5)
    n = 60000
    low = torch.randint(0, 255, (n, 1), generator=gen)
    exponent = (low - torch.randint(0, 14, (n, 32), generator=gen)).clamp(0, 254)
    bits = (torch.randint(0, 2, (n, 32), generator=gen) << 31) | (exponent << 23) | torch.randint(0, 1 << 23, (n, 32), generator=gen)
    x = torch.where(bits >= 1 << 31, bits - (1 << 32), bits).to(torch.int32).view(torch.float32)[:, None].contiguous()
    codes, scales = ref.encode(fmt, x.double())
    row = codes.shape[-1]
    dev_codes, dev_scales = torch.zeros(n, 1, 1, row, dtype=torch.uint8, device="cuda"), torch.zeros(n, 1, 1, 1, dtype=torch.uint8, device="cuda")
    hip.Cache(fmt, 1, 32, 1, n, [dev_codes], [dev_scales]).write("f32", [x.cuda()], torch.arange(n, device="cuda"), n)
    torch.cuda.synchronize()
    assert torch.equal(dev_scales.cpu().view(n, 1, 1), scales)
    off = (dev_codes.cpu().view(n, row) != codes.view(n, row)).any(-1)
    assert not bool(off.any()), "%d of %d blocks, first %s" % (int(off.sum()), n, x[off][0])
