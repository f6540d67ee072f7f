"""pccl_hip_cache_write and pccl_hip_cache_read against the restatement of cache_reference.py, bit for bit: every format and
type, heads of odd sizes, layouts, pages that end inside a workgroup's share, slots that name nothing, values at the formats' edges."""
import pytest

import cache_reference as ref

pytestmark = pytest.mark.gpu

FORMATS = ["f8e4m3", "f8e5m2", "i8", "f4e2m1"]
DTYPES = ["f32", "bf16", "f16"]


class Pages:
    """n tensors of codes and scales on the device and their copies on the host, filled with a pattern."""

    def __init__(self, torch, hip, fmt, heads, dim, page, pages, n=2, layout="token", seed=1):
        gen = torch.Generator().manual_seed(seed)
        row, blocks = hip.Cache.row_bytes(fmt, dim)
        self.shape = (pages, page, heads)
        self.codes, self.scales, self.strides = [], [], []
        for size in (row, blocks):
            pad = 3 if layout == "gaps" else 0
            if layout == "head":   # heads outside of tokens
                s = (page * heads * size, size, page * size)
            else:
                s = (page * (heads * (size + pad) + pad) + pad, heads * (size + pad) + pad, size + pad)
            self.strides.append(s)
            for _ in range(n):
                raw = torch.randint(0, 256, (max(1, pages * max(s) + 64),), generator=gen, dtype=torch.uint8)
                (self.codes if size is row and len(self.strides) == 1 else self.scales).append(raw)
        self.sizes = (row, blocks)
        self.dev_codes, self.dev_scales = [x.cuda() for x in self.codes], [x.cuda() for x in self.scales]
        self.cache = hip.Cache(fmt, heads, dim, page, pages, self.dev_codes, self.dev_scales, *self.strides)

    def view(self, raw, which):
        """[pages, tokens, heads, bytes] of a host copy"""
        return raw.as_strided((*self.shape, self.sizes[which]), (*self.strides[which], 1))


def source(torch, gen, dtype, tokens, heads, dim):
    """Ordinary values with blocks of every kind that a format finds hard among them."""
    x = torch.randn(tokens, heads, dim, generator=gen, dtype=torch.float64) * torch.exp(2 * torch.randn(tokens, heads, 1, generator=gen, dtype=torch.float64))
    t = ref.TYPES[dtype]
    info = torch.finfo(t)
    flat = x.view(-1, dim)
    kinds = [lambda v: v.zero_(), lambda v: v.fill_(-0.0), lambda v: v.mul_(info.tiny * 2), lambda v: v.mul_(info.tiny * info.eps * 40),
             lambda v: v.clamp_(-1, 1).mul_(info.max / 1.0), lambda v: v[:1].fill_(float("inf")), lambda v: v[-1:].fill_(float("nan")),
             lambda v: v.copy_((torch.randint(-512, 513, v.shape, generator=gen) / 64).double()),   # many ties
             lambda v: v.copy_((torch.randint(-127, 128, v.shape, generator=gen) / 128).double()),
             lambda v: v.copy_(torch.randint(-16, 17, v.shape, generator=gen).double() * info.tiny / 8), lambda v: v[:1].fill_(-float("inf"))]
    for k in range(flat.shape[0]):
        if k % 3 == 0:
            kinds[(k // 3) % len(kinds)](flat[k])
    return x.to(t)


@pytest.mark.parametrize("layout", ["token", "head", "gaps"])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("fmt", FORMATS)
def test_write(hip, fmt, dtype, layout):
    import torch
    gen = torch.Generator().manual_seed(FORMATS.index(fmt) * 10 + DTYPES.index(dtype))
    for heads, dim, page, pages, tokens in ((1, 1, 1, 1, 1), (1, 7, 3, 4, 5), (2, 8, 4, 9, 30), (3, 31, 5, 9, 41), (2, 32, 16, 8, 100),
                                            (5, 33, 7, 30, 200), (4, 64, 16, 16, 256), (3, 72, 13, 20, 177), (1, 128, 64, 4, 256),
                                            (8, 130, 16, 9, 99), (2, 255, 1, 60, 33), (1, 1000, 2, 9, 17)):
        p = Pages(torch, hip, fmt, heads, dim, page, pages, layout=layout)
        gap = 5 if layout == "gaps" else 0  # a source with gaps between heads and tokens, off the packs' alignment
        x = [source(torch, gen, dtype, tokens, heads, dim) for _ in range(2)]
        wide = [torch.full((tokens, heads, dim + gap), 3.0, dtype=x[0].dtype, device="cuda") for _ in range(2)]
        for w, v in zip(wide, x):
            w[..., :dim] = v.cuda()
        slots = torch.randperm(pages * page, generator=gen)[:tokens].clone()
        nothing = torch.rand(tokens, generator=gen) < 0.15
        slots[nothing] = torch.tensor([-1, pages * page, -(1 << 40), 1 << 40, pages * page + 7])[torch.randint(0, 5, (int(nothing.sum()),), generator=gen)]
        p.cache.write(dtype, wide, slots.cuda(), tokens, torch.cuda.current_stream().cuda_stream, heads * (dim + gap), dim + gap)
        torch.cuda.synchronize()
        kept = (slots >= 0) & (slots < pages * page)
        at = slots[kept]
        for k in range(2):
            codes, scales = ref.encode(fmt, x[k].double())
            p.view(p.codes[k], 0)[at // page, at % page] = codes[kept]
            p.view(p.scales[k], 1)[at // page, at % page] = scales[kept]
            what = "%s %s %s heads %d dim %d tensor %d" % (fmt, dtype, layout, heads, dim, k)
            assert torch.equal(p.dev_scales[k].cpu(), p.scales[k]), "scales, " + what
            assert torch.equal(p.dev_codes[k].cpu(), p.codes[k]), "codes, " + what


@pytest.mark.parametrize("layout", ["token", "head", "gaps"])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("fmt", FORMATS)
def test_read(hip, fmt, dtype, layout):
    import torch
    gen = torch.Generator().manual_seed(100 + FORMATS.index(fmt) * 10 + DTYPES.index(dtype))
    for heads, dim, page, lengths, packed in ((1, 1, 1, [1], False), (1, 7, 3, [5, 0, 3], False), (2, 8, 4, [1, 9, 4, 8], True), (3, 31, 5, [41, 0, 12], True),
                                              (2, 32, 16, [100, 16, 17], False), (5, 33, 7, [60, 7, 8, 6], True), (4, 64, 16, [256], False),
                                              (3, 72, 13, [77, 90, 13, 1, 0], True), (8, 130, 16, [33, 60], False), (2, 255, 1, [9, 17], True), (1, 1000, 2, [17], False)):
        need = [-(-n // page) for n in lengths]
        pages = sum(need) + 2
        p = Pages(torch, hip, fmt, heads, dim, page, pages, layout=layout, seed=dim)  # every code and every scale, at random
        order, at = torch.randperm(pages, generator=gen), 0
        table = torch.full((len(lengths), max(need) + 1), -1, dtype=torch.int32)
        for s, k in enumerate(need):
            table[s, :k] = order[at:at + k].int()
            at += k
        if len(lengths) > 2 and need[2] > 1:
            table[2, 1] = pages + 5   # a page that is not there: its rows are left alone
        max_len = max(lengths)
        gap = 3 if layout == "gaps" else 0
        rows = sum(lengths) + 4 if packed else len(lengths) * max_len
        start = [sum(lengths[:s]) + 2 for s in range(len(lengths))] if packed else [s * max_len for s in range(len(lengths))]
        outs = [torch.full((rows, heads, dim + gap), 3.0, dtype=ref.TYPES[dtype], device="cuda") for _ in range(2)]
        p.cache.read(dtype, outs, table.cuda(), torch.tensor(lengths, dtype=torch.int32).cuda(), len(lengths), max_len,
                     row_start=torch.tensor(start).cuda() if packed else None, out_rows=rows, stream=torch.cuda.current_stream().cuda_stream,
                     token_stride=heads * (dim + gap), head_stride=dim + gap)
        torch.cuda.synchronize()
        for k in range(2):
            want = torch.full((rows, heads, dim + gap), 3.0, dtype=ref.TYPES[dtype])
            codes, scales = p.view(p.codes[k], 0), p.view(p.scales[k], 1)
            for s, n in enumerate(lengths):
                for t in range(n):
                    page_of = int(table[s, t // page])
                    if page_of < pages:
                        want[start[s] + t, :, :dim] = ref.decode(fmt, codes[page_of, t % page], scales[page_of, t % page], dim, dtype)
            assert ref.same(outs[k], want), "%s %s %s heads %d dim %d tensor %d" % (fmt, dtype, layout, heads, dim, k)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("fmt", FORMATS)
def test_every_code_with_every_scale(hip, fmt, dtype):
    """256 tokens with one scale byte each, every code in each of them."""
    import torch
    codes = torch.arange(256, dtype=torch.uint8).repeat(256, 1, 1).contiguous()
    dim = 256 if ref.BITS[fmt] == 8 else 512
    scales = torch.arange(256, dtype=torch.uint8)[:, None, None].expand(-1, -1, dim // 32).contiguous()
    cache = hip.Cache(fmt, 1, dim, 256, 1, [codes.cuda()], [scales.cuda()])
    out = torch.zeros(256, 1, dim, dtype=ref.TYPES[dtype], device="cuda")
    table, lengths = torch.zeros(1, 1, dtype=torch.int32, device="cuda"), torch.tensor([256], dtype=torch.int32, device="cuda")
    cache.read(dtype, [out], table, lengths, 1, 256)
    torch.cuda.synchronize()
    assert ref.same(out, ref.decode(fmt, codes, scales, dim, dtype))


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("fmt", FORMATS)
def test_every_pattern_under_scales_near_its_own(hip, fmt, dtype):
    """All 65536 patterns of a 16-bit type, 31 to a block in the order of their magnitude, each block with one element that is the
    largest of them times 1, 1.5, 2, ... 2^8 and sets the scale."""
    import torch
    t = ref.TYPES[dtype]
    bits = torch.arange(65536, dtype=torch.int32)
    order = torch.argsort((bits & 0x7fff) * 2 + (bits >> 15))
    patterns = torch.cat([bits[order], bits[order][-(-65536 % 31):]]).to(torch.int16).view(t).view(-1, 31)
    most = torch.where(torch.isfinite(patterns), patterns.double().abs(), 0.0).amax(-1)
    blocks = []
    for k in range(9):
        for f in (1.0, 1.5):
            lead = (most * f * 2.0 ** k).clamp(max=float(torch.finfo(t).max)).to(t)
            blocks.append(torch.cat([lead[:, None], patterns], 1))
    x = torch.cat(blocks)[:, None, :].contiguous()  # tokens x 1 head x 32
    n = x.shape[0]
    codes, scales = ref.encode(fmt, x.double())
    row = codes.shape[-1]
    dev_codes, dev_scales = torch.zeros(n, 1, 1, row, dtype=torch.uint8, device="cuda"), torch.zeros(n, 1, 1, 1, dtype=torch.uint8, device="cuda")
    hip.Cache(fmt, 1, 32, 1, n, [dev_codes], [dev_scales]).write(dtype, [x.cuda()], torch.arange(n, device="cuda"), n)
    torch.cuda.synchronize()
    assert torch.equal(dev_scales.cpu().view(n, 1, 1), scales)
    off = (dev_codes.cpu().view(n, row) != codes.view(n, row)).any(-1)
    assert not bool(off.any()), "%d of %d blocks, first %s" % (int(off.sum()), n, x[off][0])
