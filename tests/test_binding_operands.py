"""What the binding of the norms and the cache looks at in front of a call: numbers that their fields can't hold, and what operands that
can tell (torch tensors) say of themselves.  No GPU needed: every call is refused, or has no rows."""
import pytest

from pccl_amd import hip

A = 0x100000


def refused(f, *a, **kw):
    with pytest.raises(hip.PcclError) as e:
        f(*a, **kw)
    assert e.value.code == hip.ERR_INVALID_ARG, str(e.value)
    return str(e.value)


def test_numbers_that_their_fields_cannot_hold():
    """2^32 + n must not be taken for n."""
    make = lambda heads=2, dim=64, page=16, pages=4, **kw: hip.Cache("i8", heads, dim, page, pages, [A], [A], **kw)  # noqa: E731
    make()
    refused(make, heads=2 ** 32 + 2)
    refused(make, dim=2 ** 32 + 64, code_strides=(2048, 128, 64), scale_strides=(64, 4, 2))
    refused(make, page=2 ** 64 + 16, code_strides=(2048, 128, 64), scale_strides=(64, 4, 2))
    refused(make, pages=2 ** 64 + 4)
    refused(make, code_strides=(2048, 128, 2 ** 64 + 64))
    refused(make, scale_strides=(2 ** 64 + 64, 4, 2))
    refused(make().read, "bf16", [A], A, A, 2 ** 32, 8, table_stride=4, out_rows=8)
    refused(hip.FoldNorm("bf16", 2 ** 32 + 64).forward, [A], [A], 0)
    refused(hip.FoldNorm("bf16", 64).forward, [A], [A], 2 ** 64)


def tensors(dtype, *shape):
    import torch
    return torch.zeros(*shape, dtype=getattr(torch, dtype))


def test_rows_of_another_element_type():
    """Every row operand of every call; a list's last one too."""
    good, bad = tensors("bfloat16", 0), tensors("float32", 0)
    n = hip.FoldNorm("bf16", 64, post="rms")
    n.forward([good, good], [good, good], 0, residual=good, residual_out=good, folded=good)
    for kw in (dict(ins=[good, bad]), dict(outs=[good, bad]), dict(residual=bad), dict(residual_out=bad), dict(folded=bad)):
        assert "float32" in refused(n.forward, kw.pop("ins", [good, good]), kw.pop("outs", [good]), 0, **kw)
    n.backward([good], [good], [good], 0, residual_out=good, grad_residual_out=good, grad_residual=good)
    for kw in (dict(ins=[bad]), dict(grad_outs=[good, bad]), dict(grad_ins=[bad]), dict(residual_out=bad), dict(grad_residual_out=bad),
               dict(grad_residual=bad)):
        refused(n.backward, kw.pop("ins", [good]), kw.pop("grad_outs", [good]), kw.pop("grad_ins", [good]), 0, **kw)
    c = hip.Cache("i8", 2, 64, 16, 4, [A, A], [A, A])
    index = tensors("int32", 0)
    c.write("bf16", [good, good], index.long(), 0)
    refused(c.write, "bf16", [good, bad], index.long(), 0)
    refused(c.write, "f32", [good, good], index.long(), 0)
    c.read("bf16", [good, good], index, index, 0, 8, table_stride=4)
    refused(c.read, "bf16", [good, bad], index, index, 0, 8, table_stride=4)


def test_raw_bits_and_addresses_pass():
    raw, raw_bytes = tensors("int16", 0), tensors("uint8", 0)

    class Buffer:  # (says where it is, not what it holds)
        def data_ptr(self):
            return A

    hip.FoldNorm("bf16", 64).forward([raw, A, Buffer()], [Buffer(), raw_bytes], 0, residual=raw)
    hip.FoldNorm("f32", 64).forward([raw_bytes], [raw], 0)
    assert "64 elements" in refused(hip.FoldNorm, "f32", 64, pre_weight=tensors("uint8", 255))
    assert "device memory" in refused(hip.FoldNorm, "f32", 64, pre_weight=tensors("uint8", 256))
    refused(hip.FoldNorm("bf16", 64).forward, [tensors("float16", 0)], [A], 0)


def test_parameters():
    """bf16 rows with binary32 weights are named by param_dtype; without it the weights were read as bf16."""
    make = hip.FoldNorm
    for what in ("post_weight", "post_bias", "pre_weight", "pre_bias"):
        assert "float32" in refused(make, "bf16", 64, post="rms", **{what: tensors("float32", 64)})
        refused(make, "bf16", 64, post="rms", param_dtype="f32", **{what: tensors("bfloat16", 64)})
        refused(make, "f32", 64, post="rms", **{what: tensors("float64", 64)})
        assert "64 elements" in refused(make, "f32", 64, post="rms", **{what: tensors("float32", 63)})
        assert "side by side" in refused(make, "f32", 64, post="rms", **{what: tensors("float32", 128)[::2]})
        assert "side by side" in refused(make, "f32", 64, post="rms", **{what: tensors("float32", 1).expand(64)})
    n = make("bf16", 64, post="rms", param_dtype="f32", pre_weight=A, post_weight=A)
    n.forward([A], [A], 0, gate=tensors("float32", 0), gate_rows=1)
    refused(n.forward, [A], [A], 0, gate=tensors("bfloat16", 0), gate_rows=1)
    for what in ("grad_gate", "grad_post_weight", "grad_pre_weight"):
        refused(n.backward, [A], [A], [A], 0, gate=A, gate_rows=1, **{what: tensors("bfloat16", 0)})


def test_codes_and_scales_that_are_too_short():
    pages, page, heads, dim = 3, 4, 2, 64
    make = lambda codes, scales, **kw: hip.Cache("i8", heads, dim, page, pages, [codes], [scales], **kw)  # noqa: E731
    codes, scales = pages * page * heads * dim, pages * page * heads * 2
    assert "%d are needed" % codes in refused(make, tensors("uint8", codes - 1), A)
    assert "%d are needed" % codes in refused(make, tensors("float32", codes // 4 - 1), A)
    assert "%d are needed" % scales in refused(make, A, tensors("uint8", scales - 1))
    padded = dict(code_strides=(page * heads * dim + 100, heads * dim, dim))
    refused(make, tensors("uint8", codes + 199), A, **padded)
    # whatever the view says, what counts is the memory behind its first element
    both = tensors("uint8", pages, 2, page, heads, dim)
    kv = dict(code_strides=(2 * page * heads * dim, heads * dim, dim))
    for view in (both[:, 0], both[:, 1]):
        assert "device memory" in refused(make, view, A, **kv)
    refused(make, both.flatten()[page * heads * dim + 1:], A, **kv)


def test_host_memory():
    """A tensor that the GPU can't reach is refused and not read."""
    x, w = tensors("bfloat16", 2, 64), tensors("bfloat16", 64)
    n = hip.FoldNorm("bf16", 64)
    for call in (lambda: n.forward([x], [A], 2), lambda: n.forward([A], [A, x], 2), lambda: n.forward([A], [A], 2, residual=x),
                 lambda: n.forward([A], [A], 2, gate=w, gate_rows=2), lambda: n.backward([x], [A], [A], 2, residual_out=A),
                 lambda: hip.FoldNorm("bf16", 64, pre_weight=w),
                 lambda: hip.Cache("i8", 1, 32, 1, 1, [tensors("uint8", 32)], [A]), lambda: hip.Cache("i8", 1, 32, 1, 1, [A], [tensors("uint8", 1)])):
        assert "device memory" in refused(call)
    c = hip.Cache("i8", 1, 64, 16, 4, [A], [A])
    slots, lengths, table = tensors("int64", 2), tensors("int32", 1), tensors("int32", 1, 4)
    for call in (lambda: c.write("bf16", [A], slots, 2), lambda: c.write("bf16", [x], A, 2), lambda: c.read("bf16", [x], A, A, 1, 8, table_stride=4),
                 lambda: c.read("bf16", [A], table, A, 1, 8), lambda: c.read("bf16", [A], A, lengths, 1, 8, table_stride=4),
                 lambda: c.read("bf16", [A], A, A, 1, 8, table_stride=4, row_start=slots, out_rows=8)):
        assert "device memory" in refused(call)


def test_workspace():
    n = hip.FoldNorm("bf16", 64, pre_weight=A)
    back = lambda **kw: n.backward([A], [A], [A], 2, residual_out=A, grad_pre_weight=A, **kw)  # noqa: E731
    assert "workspace of 0 bytes" in refused(back, workspace=A)  # (an address can't tell its size)
    assert "workspace of 16 bytes" in refused(back, workspace=A, workspace_bytes=16)
    assert "device memory" in refused(back, workspace=tensors("uint8", 1 << 20))
    assert "of a buffer of 0" in refused(back, workspace=tensors("uint8", 0), workspace_bytes=1 << 20)


@pytest.mark.parametrize("stream", [0, 1, 2])
def test_default_streams(stream):
    """The default streams' handles (null, hipStreamLegacy, hipStreamPerThread) are no addresses: nothing is asked about them."""
    hip.FoldNorm("bf16", 64).forward([A], [A], 0, stream=stream)
    hip.FoldNorm("bf16", 64).backward([A], [A], [A], 0, residual_out=A, stream=stream)
    c = hip.Cache("i8", 1, 32, 1, 1, [A], [A])
    c.write("bf16", [A], A, 0, stream=stream)
    c.read("bf16", [A], A, A, 0, 8, table_stride=1, stream=stream)


def test_operands_stacked_in_one_tensor():
    """A tensor of partial outputs, copies or caches stands for the list of its first dimension."""
    two = tensors("bfloat16", 2, 0)
    n = hip.FoldNorm("bf16", 64, post="rms")
    n.forward(two, two, 0)
    n.backward(two, two, two, 0, residual_out=two[0])
    refused(n.forward, tensors("float32", 2, 0), two, 0)
    refused(n.forward, two, tensors("bfloat16", 9, 0), 0)
    raw = tensors("uint8", 2, 0)
    c = hip.Cache("i8", 1, 32, 1, 0, raw, raw)
    c.write("bf16", two, A, 0)
    c.read("bf16", two, A, A, 0, 8, table_stride=1)


def test_codes_that_their_fields_cannot_hold():
    refused(hip.FoldNorm, 2 ** 40, 64)
    refused(hip.FoldNorm, "bf16", 64, post=2 ** 33)
