"""ctypes binding of ``libpccl_hip.so`` (C ABI declared in ``include/pccl_hip.h``).

Operands are raw device addresses; anything with ``data_ptr()`` (a torch tensor) is
accepted in their place.  Every call raises :class:`PcclError` on a non-zero return
code, carrying the library's error text.
"""
import ctypes
import os
import struct
import sys

_HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(_HERE, "lib", "libpccl_hip.so")

# codes of include/pccl_hip.h
F32, I32, BF16, F16, F8E4M3, F8E5M2, F64, U32 = 0, 1, 2, 3, 4, 5, 6, 7
SUM, PROD, MIN, MAX = 0, 1, 2, 3
COPY, REDUCE, NOTIFY, GET_NOTIFIED = 0, 1, 2, 3
DTYPES = {"f32": F32, "i32": I32, "bf16": BF16, "f16": F16, "f8e4m3": F8E4M3, "f8e5m2": F8E5M2, "f64": F64, "u32": U32}
COMPUTES = {"sum": SUM, "prod": PROD, "min": MIN, "max": MAX}
ELEM_BYTES = {F32: 4, I32: 4, BF16: 2, F16: 2, F8E4M3: 1, F8E5M2: 1, F64: 8, U32: 4}

OK = 0
ERR_INVALID_ARG, ERR_UNSUPPORTED, ERR_HIP, ERR_NO_DEVICE = -1, -2, -3, -4
ERR_NOMEM, ERR_MISALIGNED, ERR_GRAPH = -5, -6, -7

MAX_INPUTS = 8
MAX_OUTPUTS = 8


NORM_NONE, NORM_RMS, NORM_LAYER = 0, 1, 2
NORMS = {"none": NORM_NONE, "rms": NORM_RMS, "layer": NORM_LAYER}
NORM_MAX_WIDTH = 16384
CACHE_F8E4M3, CACHE_F8E5M2, CACHE_I8, CACHE_F4E2M1 = 0, 1, 2, 3
CACHE_FORMATS = {"f8e4m3": CACHE_F8E4M3, "f8e5m2": CACHE_F8E5M2, "i8": CACHE_I8, "f4e2m1": CACHE_F4E2M1}
CACHE_MAX_TENSORS = 8
CACHE_BLOCK = 32


class PcclError(RuntimeError):
    def __init__(self, code, text):
        super().__init__("pccl_hip error %d: %s" % (code, text))
        self.code = code


class OpDesc(ctypes.Structure):
    """struct pccl_op_desc"""
    _fields_ = [
        ("op_uid", ctypes.c_int),
        ("primitive", ctypes.c_ubyte),
        ("dtype", ctypes.c_ubyte),
        ("compute", ctypes.c_ubyte),
        ("n_in", ctypes.c_ubyte),
        ("n_out", ctypes.c_ubyte),
        ("reserved", ctypes.c_ubyte),
        ("signal_parts", ctypes.c_ushort),
        ("ins", ctypes.c_void_p * MAX_INPUTS),
        ("outs", ctypes.c_void_p * MAX_OUTPUTS),
        ("count", ctypes.c_long),
        ("n_deps", ctypes.c_int),
        ("deps", ctypes.POINTER(ctypes.c_int)),
    ]


# struct pccl_fold_norm_desc and struct pccl_fold_norm_grads, packed in one go for each call (field by field through ctypes costs as
# much as the launch): kinds and settings, which the layer packs once; the last of those, n_in, n_out, rows, width; weights and biases;
# gate; ins; residual; residual_out; folded; outs
_FOLD_NORM_HEAD, _FOLD_NORM_DESC = struct.Struct("@4i4f"), struct.Struct("@f3i2l 4P P2l 8Pl Pl Pl Pl 8Pl")
# grad_outs; grad_residual_out; grad_ins, n_grad_in; grad_residual; grad_gate; gradients of weights and biases; workspace
_FOLD_NORM_GRADS = struct.Struct("@8Pl Pl 8P2il Pl Pl 4P Pl")
_POINTERS = struct.Struct("@8P")


class CacheDesc(ctypes.Structure):
    """struct pccl_cache_desc"""
    _fields_ = [
        ("format", ctypes.c_int), ("n_tensors", ctypes.c_int), ("heads", ctypes.c_int), ("head_dim", ctypes.c_int),
        ("page_tokens", ctypes.c_long), ("n_pages", ctypes.c_long),
        ("codes", ctypes.c_void_p * CACHE_MAX_TENSORS),
        ("code_page", ctypes.c_long), ("code_token", ctypes.c_long), ("code_head", ctypes.c_long),
        ("scales", ctypes.c_void_p * CACHE_MAX_TENSORS),
        ("scale_page", ctypes.c_long), ("scale_token", ctypes.c_long), ("scale_head", ctypes.c_long),
    ]


_lib = None


def lib():
    """Loads the library on first use; no fallback when it is missing."""
    global _lib
    if _lib is None:
        if not os.path.exists(LIB_PATH):
            raise RuntimeError(
                "%s is missing: build it with `python -c 'import __graft_entry__ as g; g.build()'` "
                "(there is no CPU fallback)" % LIB_PATH)
        L = ctypes.CDLL(LIB_PATH, mode=ctypes.RTLD_GLOBAL)
        vp, ci, cl = ctypes.c_void_p, ctypes.c_int, ctypes.c_long
        L.pccl_hip_device_count.argtypes = [ctypes.POINTER(ci)]
        L.pccl_hip_device_info.argtypes = [ctypes.POINTER(ci), ctypes.POINTER(cl), ctypes.c_char_p, ci]
        L.pccl_hip_set_executor_id.argtypes = [ci]
        L.pccl_hip_alloc.argtypes = [ctypes.POINTER(vp), cl]
        L.pccl_hip_free.argtypes = [vp]
        L.pccl_hip_reduce_copy.argtypes = [ci, ci, ctypes.POINTER(vp), ci, ctypes.POINTER(vp), ci, cl, vp]
        L.pccl_hip_accumulate.argtypes = [ci, ci, vp, ctypes.POINTER(vp), ci, cl, vp]
        L.pccl_hip_fold_norm.argtypes = [vp, vp]
        L.pccl_hip_fold_norm_backward.argtypes = [vp, vp, vp]
        L.pccl_hip_fold_norm_workspace.argtypes = [cl, cl, cl, ctypes.POINTER(cl)]
        L.pccl_hip_cache_write.argtypes = [vp, ci, vp, cl, cl, vp, cl, vp]
        L.pccl_hip_cache_read.argtypes = [vp, ci, vp, cl, cl, cl, vp, cl, vp, vp, ci, cl, vp]
        L.pccl_hip_set_tuning.argtypes = [ci, ci]
        L.pccl_hip_set_occupancy_lds.argtypes = [ci]
        L.pccl_hip_set_unroll.argtypes = [ci]
        L.pccl_hip_set_rotation.argtypes = [ci]
        L.pccl_hip_set_slice_bytes.argtypes = [cl]
        L.pccl_hip_graph_create.argtypes = [ctypes.POINTER(OpDesc), ci, cl, ctypes.POINTER(vp)]
        L.pccl_hip_graph_run_static.argtypes = [ctypes.POINTER(OpDesc), ci, cl, vp, ctypes.POINTER(ctypes.c_uint),
                                                ctypes.POINTER(ctypes.c_uint)]
        L.pccl_hip_graph_run.argtypes = [vp, vp]
        L.pccl_hip_graph_status.argtypes = [vp, vp, ctypes.POINTER(ctypes.c_uint), ctypes.POINTER(ctypes.c_uint)]
        L.pccl_hip_graph_rebind.argtypes = [vp, vp, vp, cl, vp]
        L.pccl_hip_graph_info.argtypes = [vp, ctypes.POINTER(vp), ctypes.POINTER(ci), ctypes.POINTER(ci)]
        L.pccl_hip_graph_launch_kind.argtypes = [vp, ctypes.POINTER(ci)]
        L.pccl_hip_classify_dependencies.argtypes = [ctypes.POINTER(OpDesc), ci, ctypes.POINTER(ci), vp]
        L.pccl_hip_plan_chains.argtypes = [ctypes.POINTER(OpDesc), ci, ctypes.POINTER(ci), ci, ctypes.POINTER(ci)]
        L.pccl_hip_plan_signals.argtypes = [ctypes.POINTER(OpDesc), ci, ctypes.POINTER(ci), ctypes.POINTER(ci)]
        L.pccl_hip_graph_dependency_kinds.argtypes = [vp, vp, ctypes.c_long, ctypes.POINTER(ctypes.c_long)]
        L.pccl_hip_graph_trace.argtypes = [vp, ci]
        L.pccl_hip_graph_read_trace.argtypes = [vp, vp, vp, ctypes.c_long, ctypes.POINTER(ctypes.c_long)]
        L.pccl_hip_graph_next_signal_base.argtypes = [vp, ctypes.POINTER(ctypes.c_uint)]
        L.pccl_hip_graph_set_spin_limit.argtypes = [vp, ctypes.c_uint]
        L.pccl_hip_graph_destroy.argtypes = [vp]
        for name in ("pccl_hip_last_error", "pccl_hip_version"):
            getattr(L, name).restype = ctypes.c_char_p
            getattr(L, name).argtypes = []
        _lib = L
    return _lib


def _check(rc):
    if rc:
        raise PcclError(rc, lib().pccl_hip_last_error().decode())


def _addr(x):
    if x is None:
        return None
    return int(x.data_ptr()) if hasattr(x, "data_ptr") else int(x)


def _code(table, x):
    return table[x] if isinstance(x, str) else int(x)


def version():
    return lib().pccl_hip_version().decode()


def device_count():
    n = ctypes.c_int(0)
    _check(lib().pccl_hip_device_count(ctypes.byref(n)))
    return n.value


def device_info():
    cus, mem = ctypes.c_int(0), ctypes.c_long(0)
    name = ctypes.create_string_buffer(256)
    _check(lib().pccl_hip_device_info(ctypes.byref(cus), ctypes.byref(mem), name, 256))
    return {"compute_units": cus.value, "hbm_bytes": mem.value, "name": name.value.decode()}


def set_executor_id(ident):
    """The registry id the device image's executor fields carry (pccl_hip_set_executor_id)."""
    _check(lib().pccl_hip_set_executor_id(ident))


def alloc(nbytes):
    p = ctypes.c_void_p(None)
    _check(lib().pccl_hip_alloc(ctypes.byref(p), nbytes))
    return p.value


def free(ptr):
    _check(lib().pccl_hip_free(ctypes.c_void_p(ptr)))


def set_rotation(rotate=-1):
    _check(lib().pccl_hip_set_rotation(rotate))


def set_slice_bytes(nbytes=0):
    """Longest stretch of an operand that one launch covers (0: the built-in 32 GiB)."""
    _check(lib().pccl_hip_set_slice_bytes(nbytes))


def set_tuning(workgroups_per_cu=0, cache_treatment=-1):
    _check(lib().pccl_hip_set_tuning(workgroups_per_cu, cache_treatment))


def set_occupancy_lds(lds_bytes=-1):
    _check(lib().pccl_hip_set_occupancy_lds(lds_bytes))


def set_unroll(unroll=-1):
    _check(lib().pccl_hip_set_unroll(unroll))


def reduce_copy(dtype, compute, ins, outs, count, stream=None):
    """One reduce-copy launch: outs[j][:count] = fold(compute, ins[0][:count], ...)."""
    n_in, n_out = len(ins), len(outs)
    a_in = (ctypes.c_void_p * max(n_in, 1))(*[_addr(x) for x in ins])
    a_out = (ctypes.c_void_p * max(n_out, 1))(*[_addr(x) for x in outs])
    _check(lib().pccl_hip_reduce_copy(_code(DTYPES, dtype), _code(COMPUTES, compute), a_in, n_in,
                                      a_out, n_out, count, ctypes.c_void_p(_addr(stream))))


def accumulate(dtype, compute, src, outs, count, stream=None):
    """outs[j][:count] = compute(outs[j][:count], src[:count]) for every j, reading src once."""
    a_out = (ctypes.c_void_p * max(len(outs), 1))(*[_addr(x) for x in outs])
    _check(lib().pccl_hip_accumulate(_code(DTYPES, dtype), _code(COMPUTES, compute), ctypes.c_void_p(_addr(src)), a_out,
                                     len(outs), count, ctypes.c_void_p(_addr(stream))))


_ZEROS = [0] * 8
_PADS = [[0] * (8 - n) for n in range(9)]  # what fills a list of n up to the fixed array of its field


def _at(x):
    """Address of an operand, 0 for none."""
    if x is None:
        return 0
    if type(x) is int:
        return x
    try:
        return x.data_ptr()
    except AttributeError:
        return int(x)


# Element types as torch names them
_TORCH = {F32: "float32", I32: "int32", BF16: "bfloat16", F16: "float16", F8E4M3: "float8_e4m3fn", F8E5M2: "float8_e5m2", F64: "float64", U32: "uint32"}


def _kind(code):
    """torch's object for a dtype code; None where there is none, or no torch (nor tensors) so far."""
    return getattr(sys.modules.get("torch"), _TORCH.get(code, ""), None)


def _on_device(x, what):
    """Refuses a tensor that the GPU can't reach (it would fault); pinned host memory it can."""
    if not x.is_cuda and x.numel() and not x.is_pinned():
        raise PcclError(ERR_INVALID_ARG, "%s: a tensor on %s, device memory is needed" % (what, x.device))


def _check_tensor(x, code, what):
    """Refuses a tensor of numbers of another type than `code`'s (read as those they would be garbage, and could end before the last row) or
    outside of the GPU's memory.  Whole numbers pass, whatever their size: a buffer of raw bytes.  Operands that are no tensors are taken at
    their word."""
    kind, torch = getattr(x, "dtype", None), sys.modules.get("torch")
    if torch is None or not isinstance(kind, torch.dtype):
        return
    if code in ELEM_BYTES and kind is not _kind(code) and (kind.is_floating_point or kind.is_complex):
        raise PcclError(ERR_INVALID_ARG, "%s: elements are %s, not %s" % (what, kind, _TORCH[code]))
    _on_device(x, what)


def _typed(x, kind, code, what):
    """Address of an operand with elements of dtype `code`, 0 for none."""
    try:
        if x.dtype is kind and x.is_cuda:
            return x.data_ptr()
        _check_tensor(x, code, what)
    except AttributeError:
        pass
    return _at(x)


def _many(x, most, kind, code, what):
    """Addresses of a list of operands with elements of dtype `code`, padded to the fixed array that they go to.  Of tensors that are all
    of that type the first one's device stands for theirs: each look costs a small call 0.05 us (8 -> 8 rows of a decoding step 5.7 us with
    no looks, 6.0 with these, 6.4 with every device)."""
    n = len(x)
    try:
        at = [t.data_ptr() for t in x if t.dtype is kind]
        fine = len(at) == n and (n == 0 or x[0].is_cuda)
    except AttributeError:
        fine = False
    if not fine:
        at = [_typed(t, kind, code, what) for t in x]
    if n > most:
        raise PcclError(ERR_INVALID_ARG, "%d %s, at most %d" % (n, what, most))
    return at + _PADS[n]


def _room(x, extent, what):
    """Address of a buffer of `extent` bytes; of one that can tell (a torch tensor), whether its memory goes that far is checked, however
    it is viewed."""
    if x is not None and type(x) is not int and hasattr(x, "untyped_storage"):
        storage, at = x.untyped_storage(), x.data_ptr()
        room = storage.data_ptr() + storage.nbytes() - at if at else 0
        if room < extent:
            raise PcclError(ERR_INVALID_ARG, "%s: %d bytes, %d are needed" % (what, room, extent))
        _on_device(x, what)
    return _at(x)


def _index(x, kind, itemsize, count, what):
    """Address of a device array of whole numbers; of one that can tell (a torch tensor), size and order are checked."""
    if x is None or type(x) is int:
        return x or 0
    if hasattr(x, "element_size"):
        if x.dtype is kind and x.numel() >= count and x.is_contiguous() and x.is_cuda:
            return x.data_ptr()
        if x.element_size() != itemsize or x.numel() < count:
            raise PcclError(ERR_INVALID_ARG, "%s: %d entries of %d bytes, %d of %d are needed" % (what, x.numel(), x.element_size(), count, itemsize))
        if not x.is_contiguous():  # (an expanded one has fewer entries in memory than it counts)
            raise PcclError(ERR_INVALID_ARG, "%s: entries must lie side by side" % what)
        _on_device(x, what)
    return _at(x)


class FoldNorm:
    """The norms around a block, fused with the fold of its partial outputs, its gate and its residual scale
    (pccl_hip_fold_norm); `width` elements a row:

        y = fold(ins)   n = post(y)   r = residual_scale * residual + block_scale * gate * n   h = pre(r)

    post, pre: "none", "rms" or "layer"; weights and biases are device vectors of `param_dtype` (by default the
    rows' dtype) and may be None; `weight_offset` is added to the weights.  The object holds these settings and
    a reference to each parameter, nothing of a call: it may be used from several threads at once."""

    def __init__(self, dtype, width, post="none", pre="rms", param_dtype=None, post_weight=None, post_bias=None, pre_weight=None,
                 pre_bias=None, post_eps=1e-6, pre_eps=1e-6, weight_offset=0.0, residual_scale=1.0, block_scale=1.0):
        self.width = width
        self._params = (post_weight, post_bias, pre_weight, pre_bias)
        dtype = _code(DTYPES, dtype)
        params = dtype if param_dtype is None else _code(DTYPES, param_dtype)
        for x, what in zip(self._params, ("post_weight", "post_bias", "pre_weight", "pre_bias")):
            if x is not None and hasattr(x, "is_contiguous") and (x.numel() * x.element_size() < width * ELEM_BYTES.get(params, 0) or not x.is_contiguous()):
                raise PcclError(ERR_INVALID_ARG, "%s: %d elements side by side are needed" % (what, width))
            _check_tensor(x, params, what)
        self._addresses = [getattr(p, "data_ptr", None) or int(p or 0).__index__ for p in self._params]  # (called anew for each call)
        self._rows, self._vectors = (_kind(dtype), dtype), (_kind(params), params)
        *settings, self._block_scale = (ctypes.c_float(x).value for x in (post_eps, pre_eps, weight_offset, residual_scale, block_scale))
        try:
            self._head = _FOLD_NORM_HEAD.pack(dtype, params, _code(NORMS, post), _code(NORMS, pre), *settings)
        except struct.error as e:  # a code that its field cannot hold
            raise PcclError(ERR_INVALID_ARG, str(e)) from None

    def forward(self, ins, outs, rows, residual=None, residual_out=None, folded=None, gate=None, gate_rows=0, stream=None,
                in_stride=None, residual_stride=None, residual_out_stride=None, folded_stride=None, gate_stride=None, out_stride=None):
        """h to every buffer of `outs` (none: h is not computed), r to `residual_out`, y to `folded`, where given.  The gate
        has one row for every `gate_rows` rows.  Strides in elements from row to row, by default the width.  Of a torch tensor the element type
        is checked; how far it goes is up to the caller, as with reduce_copy."""
        w, (kind, code), (p0, p1, p2, p3) = self.width, self._rows, self._addresses
        try:
            d = self._head + _FOLD_NORM_DESC.pack(
                self._block_scale, len(ins), len(outs), 0, rows, w, p0(), p1(), p2(), p3(), 0 if gate is None else _typed(gate, *self._vectors, "gate"),
                w if gate_stride is None else gate_stride, gate_rows, *_many(ins, MAX_INPUTS, kind, code, "inputs"),
                w if in_stride is None else in_stride, 0 if residual is None else _typed(residual, kind, code, "residual"),
                w if residual_stride is None else residual_stride, 0 if residual_out is None else _typed(residual_out, kind, code, "residual_out"),
                w if residual_out_stride is None else residual_out_stride, 0 if folded is None else _typed(folded, kind, code, "folded"),
                w if folded_stride is None else folded_stride, *_many(outs, MAX_OUTPUTS, kind, code, "outputs"), w if out_stride is None else out_stride)
        except struct.error as e:  # a number that its field cannot hold
            raise PcclError(ERR_INVALID_ARG, str(e)) from None
        rc = (_lib or lib()).pccl_hip_fold_norm(d, stream if type(stream) is int else _at(stream))
        if rc:
            _check(rc)

    def workspace_bytes(self, rows, gate_rows=0):
        """Bytes of workspace that backward needs for this many rows (gate_rows = 0: no gate)."""
        n = ctypes.c_long(0)
        _check(lib().pccl_hip_fold_norm_workspace(rows, self.width, gate_rows, ctypes.byref(n)))
        return n.value

    def backward(self, ins, grad_outs, grad_ins, rows, residual_out=None, grad_residual_out=None, grad_residual=None, gate=None,
                 gate_rows=0, grad_gate=None, grad_post_weight=None, grad_post_bias=None, grad_pre_weight=None, grad_pre_bias=None,
                 workspace=None, workspace_bytes=None, stream=None, in_stride=None, residual_out_stride=None, gate_stride=None,
                 grad_out_stride=None, grad_residual_out_stride=None, grad_in_stride=None, grad_residual_stride=None, grad_gate_stride=None):
        """Gradients (pccl_hip_fold_norm_backward).  ins: the block's partial outputs again, or [folded]; residual_out: r of
        the forward pass; grad_outs: the partial gradients of h, folded here; grad_residual_out: the gradient of r from
        further on.  Written where given: grad_ins (each the gradient of y), grad_residual, grad_gate and those of the
        parameters.  workspace: a buffer of workspace_bytes(rows, gate_rows), its size taken from the buffer where it can
        tell (a torch tensor), else from the argument; no reference is kept, and it must live until the work on `stream` is done
        (torch: record_stream, or keep it)."""
        w, (kind, code), vectors, (p0, p1, p2, p3) = self.width, self._rows, self._vectors, self._addresses
        if workspace is not None and type(workspace) is not int and hasattr(workspace, "element_size"):
            _on_device(workspace, "workspace")
            room = workspace.numel() * workspace.element_size()
            if workspace_bytes is None:
                workspace_bytes = room
            elif workspace_bytes > room:
                raise PcclError(ERR_INVALID_ARG, "workspace_bytes %d of a buffer of %d" % (workspace_bytes, room))
        try:
            d = self._head + _FOLD_NORM_DESC.pack(
                self._block_scale, len(ins), len(grad_outs), 0, rows, w, p0(), p1(), p2(), p3(), 0 if gate is None else _typed(gate, *vectors, "gate"),
                w if gate_stride is None else gate_stride, gate_rows, *_many(ins, MAX_INPUTS, kind, code, "inputs"),
                w if in_stride is None else in_stride, 0, 0, 0 if residual_out is None else _typed(residual_out, kind, code, "residual_out"),
                w if residual_out_stride is None else residual_out_stride, 0, 0, *_ZEROS, 0)
            g = _FOLD_NORM_GRADS.pack(
                *_many(grad_outs, MAX_OUTPUTS, kind, code, "gradients of the outputs"), w if grad_out_stride is None else grad_out_stride,
                0 if grad_residual_out is None else _typed(grad_residual_out, kind, code, "grad_residual_out"),
                w if grad_residual_out_stride is None else grad_residual_out_stride,
                *_many(grad_ins, MAX_INPUTS, kind, code, "gradients of the inputs"), len(grad_ins), 0, w if grad_in_stride is None else grad_in_stride,
                0 if grad_residual is None else _typed(grad_residual, kind, code, "grad_residual"),
                w if grad_residual_stride is None else grad_residual_stride,
                0 if grad_gate is None else _typed(grad_gate, *vectors, "grad_gate"), w if grad_gate_stride is None else grad_gate_stride,
                0 if grad_post_weight is None else _typed(grad_post_weight, *vectors, "grad_post_weight"),
                0 if grad_post_bias is None else _typed(grad_post_bias, *vectors, "grad_post_bias"),
                0 if grad_pre_weight is None else _typed(grad_pre_weight, *vectors, "grad_pre_weight"),
                0 if grad_pre_bias is None else _typed(grad_pre_bias, *vectors, "grad_pre_bias"), _at(workspace), workspace_bytes or 0)
        except struct.error as e:
            raise PcclError(ERR_INVALID_ARG, str(e)) from None
        rc = (_lib or lib()).pccl_hip_fold_norm_backward(d, g, stream if type(stream) is int else _at(stream))
        if rc:
            _check(rc)


class Cache:
    """A cache of keys and values in pages, coded in blocks of 32 elements with a shared power-of-two scale
    (pccl_cache_desc): codes and scales are one device buffer per tensor (keys, values, ...).  The layout is pages x tokens of a
    page x heads x bytes of a head unless strides in bytes, (page, token, head), say otherwise."""

    def __init__(self, fmt, heads, head_dim, page_tokens, n_pages, codes, scales, code_strides=None, scale_strides=None):
        self._keep = (list(codes), list(scales))
        self.heads, self.head_dim, self.page_tokens, self.n_pages = heads, head_dim, page_tokens, n_pages
        d = self._desc = CacheDesc()
        d.format = _code(CACHE_FORMATS, fmt)
        d.heads, d.head_dim, d.page_tokens, d.n_pages = heads, head_dim, page_tokens, n_pages
        if len(codes) != len(scales):
            raise PcclError(ERR_INVALID_ARG, "%d tensors of codes, %d of scales" % (len(codes), len(scales)))
        if len(codes) > CACHE_MAX_TENSORS:
            raise PcclError(ERR_INVALID_ARG, "%d tensors, at most %d" % (len(codes), CACHE_MAX_TENSORS))
        d.n_tensors = self.n_tensors = len(codes)
        self._kinds = {code: _kind(code) for code in (F32, BF16, F16)}
        self._whole = {size: getattr(sys.modules.get("torch"), "int%d" % (8 * size), None) for size in (4, 8)}
        self._ref = ctypes.addressof(d)  # (the description is only read from here on)
        row, blocks = self.row_bytes(fmt, head_dim)
        d.code_page, d.code_token, d.code_head = code_strides or (page_tokens * heads * row, heads * row, row)
        d.scale_page, d.scale_token, d.scale_head = scale_strides or (page_tokens * heads * blocks, heads * blocks, blocks)
        # (ctypes drops the bits that a field has no room for: 2^32 + 8 heads would be 8)
        for name, given in (("heads", heads), ("head_dim", head_dim), ("page_tokens", page_tokens), ("n_pages", n_pages),
                            *zip(("code_page", "code_token", "code_head"), code_strides or ()),
                            *zip(("scale_page", "scale_token", "scale_head"), scale_strides or ())):
            if getattr(d, name) != given:
                raise PcclError(ERR_INVALID_ARG, "%s %d does not fit its field" % (name, given))
        counts = (n_pages, page_tokens, heads)
        for to, buffers, strides, last, what in ((d.codes, codes, (d.code_page, d.code_token, d.code_head), row, "codes"),
                                                 (d.scales, scales, (d.scale_page, d.scale_token, d.scale_head), blocks, "scales")):
            extent = last + sum((n - 1) * stride for n, stride in zip(counts, strides)) if min(counts) > 0 else 0
            to[:] = [_room(x, extent, what) for x in buffers] + _ZEROS[:CACHE_MAX_TENSORS - len(buffers)]

    @staticmethod
    def row_bytes(fmt, head_dim):
        """(bytes of codes, bytes of scales) of one token's head"""
        bits = 4 if _code(CACHE_FORMATS, fmt) == CACHE_F4E2M1 else 8
        return (head_dim * bits + 7) // 8, (head_dim + CACHE_BLOCK - 1) // CACHE_BLOCK

    def _operands(self, x, code, what):
        if len(x) != self.n_tensors:
            raise PcclError(ERR_INVALID_ARG, "%d %s for %d tensors" % (len(x), what, self.n_tensors))
        return _POINTERS.pack(*_many(x, CACHE_MAX_TENSORS, self._kinds.get(code), code, what))

    def write(self, dtype, srcs, slots, tokens, stream=None, token_stride=None, head_stride=None):
        """Codes `tokens` rows of heads x head_dim elements of every source into slots[i] = page * page_tokens + token of the page
        (int64 on the device, side by side; a slot outside the cache: the row is left out).  The slots of one call must differ.  Strides in
        elements, by default those of a dense [tokens, heads, head_dim]."""
        dtype = _code(DTYPES, dtype)
        srcs = self._operands(srcs, dtype, "sources")
        head_stride = self.head_dim if head_stride is None else head_stride
        token_stride = self.heads * self.head_dim if token_stride is None else token_stride
        _check(lib().pccl_hip_cache_write(self._ref, dtype, srcs, token_stride, head_stride,
                                          _index(slots, self._whole[8], 8, tokens, "slots"), tokens, stream if type(stream) is int else _at(stream)))

    def read(self, dtype, outs, page_table, lengths, n_seq, max_len, row_start=None, out_rows=None, table_stride=None, stream=None,
             token_stride=None, head_stride=None):
        """Token t < lengths[s] of sequence s, from page page_table[s][t // page_tokens], to row row_start[s] + t of every output (of
        `out_rows` rows), or without row_start to row s * max_len + t.  page_table, lengths (int32) and row_start (int64) are on
        the device, their entries side by side; table_stride, the entries of a sequence, is by default what a dense 2-d table says.  Rows that no token goes to
        are left as they are."""
        dtype = _code(DTYPES, dtype)
        outs = self._operands(outs, dtype, "outputs")
        head_stride = self.head_dim if head_stride is None else head_stride
        token_stride = self.heads * self.head_dim if token_stride is None else token_stride
        if table_stride is None:
            if not hasattr(page_table, "shape"):
                raise PcclError(ERR_INVALID_ARG, "table_stride is needed where the page table cannot tell it")
            table_stride = page_table.shape[-1]
        if n_seq > 0x7fffffff:  # (ctypes would drop the bits above)
            raise PcclError(ERR_INVALID_ARG, "n_seq %d outside [0, 2^31)" % n_seq)
        if out_rows is None:
            if row_start is not None:
                raise PcclError(ERR_INVALID_ARG, "row_start without out_rows")
            out_rows = n_seq * max_len
        _check(lib().pccl_hip_cache_read(self._ref, dtype, outs, token_stride, head_stride, out_rows,
                                         _index(page_table, self._whole[4], 4, n_seq * table_stride, "page_table"), table_stride,
                                         _index(lengths, self._whole[4], 4, n_seq, "lengths"), _index(row_start, self._whole[8], 8, n_seq, "row_start"), n_seq, max_len,
                                         stream if type(stream) is int else _at(stream)))


def _op_descs(ops):
    """list of op dicts -> (OpDesc array, objects to keep alive while it is in use)."""
    n = len(ops)
    arr = (OpDesc * max(n, 1))()
    keep = []
    for i, o in enumerate(ops):
        d = arr[i]
        d.op_uid = i
        prim = o.get("primitive")
        if prim in (NOTIFY, GET_NOTIFIED):
            # signal op: "signal" = address of the 32-bit word, "value" = 0..65535
            d.primitive = prim
            d.n_in, d.n_out = (0, 1) if prim == NOTIFY else (1, 0)
            (d.outs if prim == NOTIFY else d.ins)[0] = _addr(o["signal"])
            d.count = o["value"]
            d.signal_parts = o.get("parts", 0)   # >= 2: a signal of that many words, one per part of the data
        else:
            n_in, n_out = len(o["ins"]), len(o["outs"])
            d.primitive = prim if prim is not None else (COPY if n_in == 1 else REDUCE)
            d.dtype = _code(DTYPES, o["dtype"])
            d.compute = _code(COMPUTES, o.get("compute", "sum"))
            d.n_in, d.n_out = n_in, n_out
            for k in range(min(n_in, MAX_INPUTS)):
                d.ins[k] = _addr(o["ins"][k])
            for k in range(min(n_out, MAX_OUTPUTS)):
                d.outs[k] = _addr(o["outs"][k])
            d.count = o["count"]
        deps = list(o.get("deps", ()))
        d.n_deps = len(deps)
        buf = (ctypes.c_int * max(len(deps), 1))(*deps)
        keep.append(buf)
        d.deps = ctypes.cast(buf, ctypes.POINTER(ctypes.c_int))
    return arr, keep


def part_elems(count, parts):
    """Elements per part of an op cut into `parts` parts (the last part may be shorter)."""
    per = (count + parts - 1) // parts
    return (per + 63) // 64 * 64


def classify_dependencies(ops, parts):
    """The executor's rule for which dependencies are met part by part, without a device:
    ops as for Graph, parts[i] = number of parts of op i.  Returns one flag per dependency
    (ops in order, dependencies in list order)."""
    arr, keep = _op_descs(ops)
    n_deps = sum(len(o.get("deps", ())) for o in ops)
    kinds = (ctypes.c_ubyte * max(n_deps, 1))()
    pa = (ctypes.c_int * max(len(ops), 1))(*parts)
    _check(lib().pccl_hip_classify_dependencies(arr, len(ops), pa, kinds))
    return list(kinds)[:n_deps]


def plan_chains(ops, parts, forward_elem_bytes):
    """The executor's chain plan for these ops (host only): per op a tuple (next op or -1, ops in the
    chain it starts or 1, one-pass flag / index of the handed-on input, first row of its operand table)."""
    arr, keep = _op_descs(ops)
    pa = (ctypes.c_int * max(len(ops), 1))(*parts)
    words = (ctypes.c_int * max(4 * len(ops), 1))()
    _check(lib().pccl_hip_plan_chains(arr, len(ops), pa, forward_elem_bytes, words))
    return [tuple(words[4 * i:4 * i + 4]) for i in range(len(ops))]


def plan_signals(ops, with_parts=False):
    """Which signal ops ride on data ops (host only): per op the index of the COPY / REDUCE that carries
    it, or -1.  with_parts: also, per op, the K of a signal op carried part by part / of the data op that is
    cut into K parts for such signals (0 otherwise)."""
    arr, keep = _op_descs(ops)
    carrier = (ctypes.c_int * max(len(ops), 1))()
    parts = (ctypes.c_int * max(len(ops), 1))()
    _check(lib().pccl_hip_plan_signals(arr, len(ops), carrier, parts if with_parts else None))
    if with_parts:
        return list(carrier[:len(ops)]), list(parts[:len(ops)])
    return list(carrier[:len(ops)])


STATIC_ARENA_BYTES = 8 << 20
TILE_AUTO = -1   # graph_create: the executor chooses between the queue and plain launches


def graph_run_static(ops, stream=None, tile_bytes=0, wait=True):
    """Runs a DAG of ops with its device state in the library's fixed per-GPU array: no device
    allocation (pccl_hip_graph_run_static).  wait=True: waits for `stream` and returns
    (completed, total); wait=False: returns None once the launch is enqueued."""
    arr, keep = _op_descs(ops)
    if not wait:
        _check(lib().pccl_hip_graph_run_static(arr, len(ops), tile_bytes, ctypes.c_void_p(_addr(stream)), None, None))
        return None
    c, t = ctypes.c_uint(0), ctypes.c_uint(0)
    _check(lib().pccl_hip_graph_run_static(arr, len(ops), tile_bytes, ctypes.c_void_p(_addr(stream)), ctypes.byref(c),
                                           ctypes.byref(t)))
    del keep
    return c.value, t.value


class Graph:
    """A DAG of COPY / REDUCE ops resident on the device, drained by one launch."""

    def __init__(self, ops, tile_bytes=0):
        """ops: list of dicts with keys dtype, compute, ins, outs, count, deps (op index list)."""
        arr, self._keep = _op_descs(ops)
        self._h = ctypes.c_void_p(None)
        _check(lib().pccl_hip_graph_create(arr, len(ops), tile_bytes, ctypes.byref(self._h)))

    def run(self, stream=None):
        _check(lib().pccl_hip_graph_run(self._h, ctypes.c_void_p(_addr(stream))))

    def status(self, stream=None):
        c, t = ctypes.c_uint(0), ctypes.c_uint(0)
        _check(lib().pccl_hip_graph_status(self._h, ctypes.c_void_p(_addr(stream)), ctypes.byref(c), ctypes.byref(t)))
        return c.value, t.value

    def rebind(self, old_base, new_base, nbytes, stream=None):
        _check(lib().pccl_hip_graph_rebind(self._h, ctypes.c_void_p(_addr(old_base)), ctypes.c_void_p(_addr(new_base)),
                                           nbytes, ctypes.c_void_p(_addr(stream))))

    def next_signal_base(self):
        b = ctypes.c_uint(0)
        _check(lib().pccl_hip_graph_next_signal_base(self._h, ctypes.byref(b)))
        return b.value

    def set_spin_limit(self, microseconds):
        """How long a wait inside the kernel may last before the run gives up (default two seconds)."""
        _check(lib().pccl_hip_graph_set_spin_limit(self._h, microseconds))

    def info(self):
        lay, nt, nw = ctypes.c_void_p(None), ctypes.c_int(0), ctypes.c_int(0)
        _check(lib().pccl_hip_graph_info(self._h, ctypes.byref(lay), ctypes.byref(nt), ctypes.byref(nw)))
        return {"device_layout": lay.value, "n_tiles": nt.value, "n_workgroups": nw.value}

    def launch_kind(self):
        """'drain' (the persistent kernel), 'wide' (one workgroup per entry), 'launches' (plain launches) or 'chains'
        (a wide launch in the shape of a direct one: a few chains that are each one fold, a workgroup per 4 KiB)."""
        kind = ctypes.c_int(0)
        _check(lib().pccl_hip_graph_launch_kind(self._h, ctypes.byref(kind)))
        return ("drain", "wide", "launches", "chains")[kind.value]

    def dependency_kinds(self):
        """One flag per dependency (ops in uid order, dependencies in list order): 1 = met part
        by part, 0 = waits for the whole predecessor."""
        n = ctypes.c_long(0)
        _check(lib().pccl_hip_graph_dependency_kinds(self._h, None, 0, ctypes.byref(n)))
        buf = (ctypes.c_ubyte * max(n.value, 1))()
        _check(lib().pccl_hip_graph_dependency_kinds(self._h, buf, n.value, ctypes.byref(n)))
        return list(buf)[:n.value]

    def trace(self, enable=True):
        """Switches the per-entry timeline on or off for the following runs."""
        _check(lib().pccl_hip_graph_trace(self._h, 1 if enable else 0))

    def read_trace(self, stream=None):
        """Timeline of the last run: uint64 array (entries, 4) in queue order; columns: what
        (op_uid | part << 32 | workgroup << 52), ticket drawn, dependencies met, part complete,
        in ticks of the device's 100 MHz clock."""
        import numpy as np
        n = ctypes.c_long(0)
        _check(lib().pccl_hip_graph_read_trace(self._h, ctypes.c_void_p(_addr(stream)), None, 0, ctypes.byref(n)))
        out = np.zeros((n.value, 4), dtype=np.uint64)
        if n.value:
            _check(lib().pccl_hip_graph_read_trace(self._h, ctypes.c_void_p(_addr(stream)), out.ctypes.data_as(ctypes.c_void_p),
                                                   n.value, ctypes.byref(n)))
        return out

    def destroy(self):
        if self._h:
            _check(lib().pccl_hip_graph_destroy(self._h))
            self._h = ctypes.c_void_p(None)

    def __del__(self):
        try:
            self.destroy()
        except Exception:
            pass
