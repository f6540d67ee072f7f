"""Cache calls that take more than one launch: more sequences than a grid has rows, more tokens than a launch's wavefronts."""
import pytest

import cache_reference as ref

pytestmark = pytest.mark.gpu


def test_read_of_70000_sequences(hip):
    import torch
    gen = torch.Generator().manual_seed(1)
    n_seq, page, pages, dim = 70000, 2, 64, 32
    codes = torch.randint(0, 256, (pages, page, 1, dim), generator=gen, dtype=torch.uint8)
    scales = torch.randint(100, 150, (pages, page, 1, 1), generator=gen, dtype=torch.uint8)
    table = torch.randint(-1, pages + 1, (n_seq, 1), generator=gen, dtype=torch.int32)
    lengths = torch.randint(0, 4, (n_seq,), generator=gen, dtype=torch.int32)  # (3: more than max_len)
    out = torch.full((n_seq * 2, dim), -7.0, device="cuda")
    hip.Cache("i8", 1, dim, page, pages, [codes.cuda()], [scales.cuda()]).read(
        "f32", [out], table.cuda(), lengths.cuda(), n_seq, 2, stream=torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    values = ref.decode("i8", codes, scales, dim, "f32")[:, :, 0]
    there = (table >= 0) & (table < pages) & (torch.arange(2) < lengths[:, None])
    want = torch.where(there[..., None], values[table[:, 0].clamp(0, pages - 1).long()], torch.tensor(-7.0))
    assert ref.same(out, want.view(n_seq * 2, dim))


def test_write_of_more_tokens_than_a_launch(hip):
    """65536 tokens a launch at this many heads (2^26 wavefronts).  Each token's row starts one element behind the one before it."""
    import torch
    gen = torch.Generator().manual_seed(2)
    heads, page, pages, tokens = 16384, 4, 3, 2 * 65536 + 5
    named = [0, 65535, 65536, 65537, 131071, 131072, tokens - 1]
    slots = torch.full((tokens,), -1, dtype=torch.int64)
    slots[named] = torch.randperm(page * pages, generator=gen)[:len(named)]
    srcs = [torch.randn(tokens - 1 + heads, generator=gen) for _ in range(2)]
    codes = [torch.full((pages * page, heads, 1), 0x5A, dtype=torch.uint8, device="cuda") for _ in srcs]
    scales = [torch.full((pages * page, heads, 1), 0x5A, dtype=torch.uint8, device="cuda") for _ in srcs]
    hip.Cache("f8e4m3", heads, 1, page, pages, codes, scales).write(
        "f32", [s.cuda() for s in srcs], slots.cuda(), tokens, token_stride=1, stream=torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    for src, c, s in zip(srcs, codes, scales):
        want_codes, want_scales = (torch.full((pages * page, heads, 1), 0x5A, dtype=torch.uint8) for _ in range(2))
        for i in named:
            want_codes[slots[i]], want_scales[slots[i]] = ref.encode("f8e4m3", src[i:i + heads, None].double())
        assert torch.equal(c.cpu(), want_codes) and torch.equal(s.cpu(), want_scales)


@pytest.mark.parametrize("boundary", [131072, 262144])
def test_read_of_more_tokens_than_a_launch(hip, boundary):
    """131072 tokens a launch at this many heads; the sequence's first row is so far below 0 that only the tokens around the boundary are
    inside the output."""
    import torch
    gen = torch.Generator().manual_seed(3)
    heads, page, pages, max_len = 65536, 512, 3, 2 * 131072 + 7
    codes = torch.randint(0, 256, (pages, page, heads, 1), generator=gen, dtype=torch.uint8)
    scales = torch.randint(100, 150, (pages, page, heads, 1), generator=gen, dtype=torch.uint8)
    table = torch.randint(0, pages, (1, -(-max_len // page)), generator=gen, dtype=torch.int32)
    lengths, out_rows = torch.tensor([max_len], dtype=torch.int32), 14
    out = torch.full((out_rows, heads), -7.0, device="cuda")
    hip.Cache("i8", heads, 1, page, pages, [codes.cuda()], [scales.cuda()]).read(
        "f32", [out], table.cuda(), lengths.cuda(), 1, max_len, row_start=torch.tensor([5 - boundary]).cuda(), out_rows=out_rows,
        stream=torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    want = torch.full((out_rows, heads), -7.0)
    for row in range(out_rows):
        t = row - (5 - boundary)
        if t < max_len:
            p = int(table[0, t // page])
            want[row] = ref.decode("i8", codes[p, t % page], scales[p, t % page], 1, "f32")[:, 0]
    assert ref.same(out, want)


@pytest.mark.parametrize("stride", [3, 7])
def test_read_under_a_bound_far_beyond_the_tables(hip, stride):
    """max_len as no bound at all: what has no page in the table takes no part in the launch."""
    import torch
    gen = torch.Generator().manual_seed(4)
    n_seq, heads, dim, page, pages = 300, 2, 40, 5, 11
    codes = torch.randint(0, 256, (pages, page, heads, dim), generator=gen, dtype=torch.uint8)
    scales = torch.randint(100, 150, (pages, page, heads, 2), generator=gen, dtype=torch.uint8)
    table = torch.randint(0, pages, (n_seq, stride), generator=gen, dtype=torch.int32)
    lengths = torch.randint(0, stride * page + 1, (n_seq,), generator=gen, dtype=torch.int32)
    starts = torch.cat([torch.zeros(1, dtype=torch.int64), lengths.long().cumsum(0)])
    rows = int(starts[-1])
    lengths[-1] = 2 ** 31 - 1  # (tokens behind the last page are not read; those that there are are the last rows)
    rows += stride * page - (rows - int(starts[-2]))
    out = torch.full((rows + 2, heads, dim), -7.0, device="cuda")
    hip.Cache("i8", heads, dim, page, pages, [codes.cuda()], [scales.cuda()]).read(
        "f32", [out], table.cuda(), lengths.cuda(), n_seq, 2 ** 31 - 1, row_start=starts[:-1].cuda(), out_rows=rows + 2,
        stream=torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    want = torch.full((rows + 2, heads, dim), -7.0)
    values = ref.decode("i8", codes, scales, dim, "f32")
    for s in range(n_seq):
        n = min(int(lengths[s]), stride * page)
        want[int(starts[s]):int(starts[s]) + n] = values[table[s].long()].flatten(0, 1)[:n]
    assert ref.same(out, want)
