"""What the norms around a block and the cache in blocks refuse, on the host, in front of any launch (no GPU needed: operands are
numbers that stand for device addresses)."""
import pytest

from pccl_amd import hip

A = 0x100000


def refused(code, f, *a, **kw):
    with pytest.raises(hip.PcclError) as e:
        f(*a, **kw)
    assert e.value.code == code, str(e.value)
    return str(e.value)


def norm(dtype="bf16", width=64, **kw):
    return hip.FoldNorm(dtype, width, **kw)


def test_norm_settings():
    f = lambda n, **kw: n.forward([A], [A], 2, **kw)  # noqa: E731
    refused(hip.ERR_UNSUPPORTED, f, norm("i32"))
    refused(hip.ERR_UNSUPPORTED, f, norm("f64"))
    refused(hip.ERR_UNSUPPORTED, f, norm("f8e4m3"))
    refused(hip.ERR_UNSUPPORTED, f, norm(param_dtype="f16"))
    refused(hip.ERR_UNSUPPORTED, f, norm("f32", param_dtype="bf16"))
    refused(hip.ERR_UNSUPPORTED, f, norm(post=3))
    refused(hip.ERR_UNSUPPORTED, f, norm(pre=-1))
    refused(hip.ERR_INVALID_ARG, f, norm(width=0))
    refused(hip.ERR_INVALID_ARG, f, norm(width=hip.NORM_MAX_WIDTH + 1))
    for eps in (0.0, -1.0, 1e-45, float("inf"), float("nan")):
        refused(hip.ERR_INVALID_ARG, f, norm(pre_eps=eps))
        refused(hip.ERR_INVALID_ARG, f, norm(post="layer", post_eps=eps))
    for kw in (dict(weight_offset=float("nan")), dict(residual_scale=float("inf")), dict(block_scale=float("-inf"))):
        refused(hip.ERR_INVALID_ARG, f, norm(**kw))
    refused(hip.ERR_INVALID_ARG, f, norm(post="none", post_weight=A))
    refused(hip.ERR_INVALID_ARG, f, norm(pre="none", pre_bias=A))
    refused(hip.ERR_MISALIGNED, f, norm(pre_weight=A + 1))
    refused(hip.ERR_MISALIGNED, f, norm(param_dtype="f32", pre_weight=A + 2))


def test_norm_operands():
    n = norm()
    refused(hip.ERR_INVALID_ARG, n.forward, [], [A], 2)
    refused(hip.ERR_INVALID_ARG, n.forward, [A] * 9, [A], 2)
    refused(hip.ERR_INVALID_ARG, n.forward, [A], [A] * 9, 2)
    refused(hip.ERR_INVALID_ARG, n.forward, [A, None], [A], 2)
    refused(hip.ERR_INVALID_ARG, n.forward, [A], [None], 2)
    refused(hip.ERR_INVALID_ARG, n.forward, [A], [A], -1)
    refused(hip.ERR_INVALID_ARG, n.forward, [A], [A], 1 << 31)
    refused(hip.ERR_MISALIGNED, n.forward, [A + 1], [A], 2)
    refused(hip.ERR_MISALIGNED, n.forward, [A], [A + 1], 2)
    refused(hip.ERR_MISALIGNED, n.forward, [A], [A], 2, residual=A + 1)
    refused(hip.ERR_INVALID_ARG, n.forward, [A], [A], 2, gate=A, gate_rows=0)
    refused(hip.ERR_INVALID_ARG, n.forward, [A], [A], 2, gate=A, gate_rows=2, gate_stride=-64)
    refused(hip.ERR_INVALID_ARG, n.forward, [A], [A], 2, in_stride=-1)
    refused(hip.ERR_INVALID_ARG, n.forward, [A], [A], 2, residual=A, residual_stride=-64)
    assert "overlap" in refused(hip.ERR_INVALID_ARG, n.forward, [A], [A], 2, out_stride=63)
    refused(hip.ERR_INVALID_ARG, n.forward, [A], [A], 2, residual_out=A, residual_out_stride=0)
    refused(hip.ERR_INVALID_ARG, n.forward, [A], [A], 2, folded=A, folded_stride=63)


def test_norm_without_rows_is_done():
    norm().forward([A], [A], 0)
    norm().forward([None], [None], 0)
    norm().backward([None], [None], [None], 0)


def test_norm_gradients():
    n = norm(post="rms", pre_weight=A, post_weight=A)
    good = dict(residual_out=A)
    refused(hip.ERR_INVALID_ARG, n.backward, [A], [A], [A], 2)                      # r is needed
    refused(hip.ERR_INVALID_ARG, n.backward, [A], [None], [A], 2, **good)
    refused(hip.ERR_INVALID_ARG, n.backward, [A], [A], [None], 2, **good)
    refused(hip.ERR_INVALID_ARG, n.backward, [A], [A] * 9, [A], 2, **good)
    refused(hip.ERR_INVALID_ARG, n.backward, [A], [A], [A] * 9, 2, **good)
    refused(hip.ERR_MISALIGNED, n.backward, [A], [A + 1], [A], 2, **good)
    refused(hip.ERR_MISALIGNED, n.backward, [A], [A], [A], 2, grad_residual_out=A + 1, **good)
    refused(hip.ERR_INVALID_ARG, n.backward, [A], [A], [A], 2, grad_in_stride=1, **good)
    refused(hip.ERR_INVALID_ARG, n.backward, [A], [A], [A], 2, grad_residual=A, grad_residual_stride=1, **good)
    refused(hip.ERR_INVALID_ARG, n.backward, [A], [A], [A], 2, grad_gate=A, **good)           # no gate
    refused(hip.ERR_INVALID_ARG, n.backward, [A], [A], [A], 2, gate=A, gate_rows=1, grad_gate=A, grad_gate_stride=1, **good)
    refused(hip.ERR_INVALID_ARG, n.backward, [A], [A], [A], 2, gate=A, gate_rows=1, grad_gate=A, **good)   # over the gate itself
    refused(hip.ERR_INVALID_ARG, n.backward, [A], [A], [A], 2, grad_pre_bias=A, **good)       # no bias
    need = n.workspace_bytes(2)
    assert "workspace" in refused(hip.ERR_INVALID_ARG, n.backward, [A], [A], [A], 2, grad_pre_weight=A, **good)
    refused(hip.ERR_INVALID_ARG, n.backward, [A], [A], [A], 2, grad_pre_weight=A, workspace=A, workspace_bytes=need - 1, **good)
    refused(hip.ERR_MISALIGNED, n.backward, [A], [A], [A], 2, grad_pre_weight=A, workspace=A + 8, workspace_bytes=need, **good)
    refused(hip.ERR_MISALIGNED, n.backward, [A], [A], [A], 2, grad_pre_weight=A + 1, workspace=A, workspace_bytes=need, **good)
    refused(hip.ERR_INVALID_ARG, n.workspace_bytes, -1)
    refused(hip.ERR_INVALID_ARG, n.workspace_bytes, 1, -1)


def cache(fmt="i8", heads=2, dim=64, page=16, pages=4, n=2, **kw):
    return hip.Cache(fmt, heads, dim, page, pages, [A] * n, [A] * n, **kw)


def test_cache_description():
    w = lambda c: c.write("bf16", [A] * c.n_tensors, A, 1)  # noqa: E731
    refused(hip.ERR_UNSUPPORTED, w, cache(4))
    refused(hip.ERR_INVALID_ARG, w, cache(heads=0))
    refused(hip.ERR_INVALID_ARG, w, cache(dim=0))
    refused(hip.ERR_INVALID_ARG, w, cache(dim=65537))
    refused(hip.ERR_INVALID_ARG, w, cache(page=0))
    refused(hip.ERR_INVALID_ARG, w, cache(pages=-1))
    refused(hip.ERR_INVALID_ARG, w, cache(page=1 << 20, pages=1 << 11))
    refused(hip.ERR_INVALID_ARG, cache, n=9)
    refused(hip.ERR_INVALID_ARG, w, cache(n=0))
    refused(hip.ERR_INVALID_ARG, hip.Cache, "i8", 1, 32, 1, 1, [A], [A, A])
    assert "overlap" in refused(hip.ERR_INVALID_ARG, w, cache(code_strides=(2048, 128, 63)))
    refused(hip.ERR_INVALID_ARG, w, cache(code_strides=(2047, 128, 64)))
    refused(hip.ERR_INVALID_ARG, w, cache(scale_strides=(64, 3, 2)))
    refused(hip.ERR_INVALID_ARG, w, cache(scale_strides=(-64, 4, 2)))
    refused(hip.ERR_INVALID_ARG, w, hip.Cache("i8", 1, 32, 1, 1, [None], [A]))


def test_cache_write():
    c = cache()
    refused(hip.ERR_UNSUPPORTED, c.write, "i32", [A, A], A, 1)
    refused(hip.ERR_INVALID_ARG, c.write, "bf16", [A], A, 1)
    refused(hip.ERR_INVALID_ARG, c.write, "bf16", [A, None], A, 1)
    refused(hip.ERR_INVALID_ARG, c.write, "bf16", [A, A], None, 1)
    refused(hip.ERR_INVALID_ARG, c.write, "bf16", [A, A], A, -1)
    refused(hip.ERR_INVALID_ARG, c.write, "bf16", [A, A], A, 1 << 31)
    refused(hip.ERR_MISALIGNED, c.write, "bf16", [A, A + 1], A, 1)
    refused(hip.ERR_MISALIGNED, c.write, "bf16", [A, A], A + 4, 1)
    refused(hip.ERR_INVALID_ARG, c.write, "bf16", [A, A], A, 1, token_stride=-1)
    refused(hip.ERR_INVALID_ARG, c.write, "bf16", [A, A], A, 1, head_stride=-1)
    refused(hip.ERR_INVALID_ARG, c.write, "bf16", [A, A], A, 1, head_stride=(1 << 40) + 1)
    refused(hip.ERR_UNSUPPORTED, c.write, "bf16", [A, A], A, 1, token_stride=1 << 31)
    refused(hip.ERR_UNSUPPORTED, cache(code_strides=(1 << 32, 128, 64)).write, "bf16", [A, A], A, 1)
    refused(hip.ERR_UNSUPPORTED, cache(scale_strides=(1 << 32, 4, 2)).write, "bf16", [A, A], A, 1)
    c.write("bf16", [A, A], A, 0)
    c.write("bf16", [None, None], None, 0)


def test_cache_index_arrays_that_tell_their_size():
    import torch
    c = cache()
    refused(hip.ERR_INVALID_ARG, c.write, "bf16", [A, A], torch.zeros(4, dtype=torch.int32), 4)
    refused(hip.ERR_INVALID_ARG, c.write, "bf16", [A, A], torch.zeros(3, dtype=torch.int64), 4)
    table, n = torch.zeros(2, 3, dtype=torch.int32), torch.zeros(2, dtype=torch.int32)
    refused(hip.ERR_INVALID_ARG, c.read, "bf16", [A, A], table.long(), n, 2, 8)
    refused(hip.ERR_INVALID_ARG, c.read, "bf16", [A, A], table, n[:1], 2, 8)
    refused(hip.ERR_INVALID_ARG, c.read, "bf16", [A, A], table, n, 3, 8)
    refused(hip.ERR_INVALID_ARG, c.read, "bf16", [A, A], table, n, 2, 8, row_start=n, out_rows=8)
    refused(hip.ERR_INVALID_ARG, c.read, "bf16", [A, A], table, n, 2, 8, row_start=n.long())


def test_cache_index_arrays_in_another_order():
    import torch
    c = cache()
    table, n, rows = torch.zeros(4, 6, dtype=torch.int32), torch.zeros(8, dtype=torch.int32), torch.zeros(8, dtype=torch.int64)
    refused(hip.ERR_INVALID_ARG, c.write, "bf16", [A, A], rows[::2], 4)
    refused(hip.ERR_INVALID_ARG, c.write, "bf16", [A, A], rows[:1].expand(4), 4)
    refused(hip.ERR_INVALID_ARG, c.read, "bf16", [A, A], table[:, :4], n, 4, 8)
    refused(hip.ERR_INVALID_ARG, c.read, "bf16", [A, A], table[:1].expand(4, 6), n, 4, 8)
    refused(hip.ERR_INVALID_ARG, c.read, "bf16", [A, A], table.t(), n, 4, 8)
    refused(hip.ERR_INVALID_ARG, c.read, "bf16", [A, A], table, n[::2], 4, 8)
    refused(hip.ERR_INVALID_ARG, c.read, "bf16", [A, A], table, n, 4, 8, row_start=rows[::2], out_rows=32)
    refused(hip.ERR_INVALID_ARG, c.read, "bf16", [A, A], A, A, 4, 8)


def test_cache_read():
    c = cache()
    r = lambda outs=(A, A), table=A, lengths=A, n=1, most=8, stride=4, **kw: c.read(  # noqa: E731
        kw.pop("dtype", "bf16"), list(outs), table, lengths, n, most, table_stride=stride, **kw)
    refused(hip.ERR_UNSUPPORTED, r, dtype="f8e4m3")
    refused(hip.ERR_INVALID_ARG, r, outs=(A,))
    refused(hip.ERR_INVALID_ARG, r, outs=(A, None))
    refused(hip.ERR_MISALIGNED, r, outs=(A, A + 1))
    refused(hip.ERR_INVALID_ARG, r, table=None)
    refused(hip.ERR_INVALID_ARG, r, lengths=None)
    refused(hip.ERR_MISALIGNED, r, table=A + 2)
    refused(hip.ERR_MISALIGNED, r, lengths=A + 2)
    refused(hip.ERR_MISALIGNED, r, row_start=A + 4, out_rows=8)
    refused(hip.ERR_INVALID_ARG, r, n=-1)
    refused(hip.ERR_INVALID_ARG, r, most=-1)
    refused(hip.ERR_INVALID_ARG, r, most=1 << 31)
    refused(hip.ERR_INVALID_ARG, r, stride=-1)
    refused(hip.ERR_INVALID_ARG, r, out_rows=-1)
    refused(hip.ERR_INVALID_ARG, r, out_rows=1 << 31)
    refused(hip.ERR_UNSUPPORTED, r, token_stride=1 << 31)
    assert "overlap" in refused(hip.ERR_INVALID_ARG, r, token_stride=127)
    refused(hip.ERR_INVALID_ARG, r, head_stride=63)
    r(n=0, table=None, lengths=None)
    r(most=0)
