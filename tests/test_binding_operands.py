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
