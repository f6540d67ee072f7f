"""Plain restatement of the norms around a block (pccl_hip_fold_norm) in 64 bits, and how far a computation in
32 bits may be from it.

Bounds.  u = 2^-24 is half a step of binary32.  A sum of a row's elements has a depth of at most 16 terms in a lane, 6 steps in
a wavefront and 16 over wavefronts, so its error is below 40 u times the sum of magnitudes; a square root's reciprocal adds
one step, every other operation half a step of its own value.  K = 64 covers what is chained between two stores of one
element: fold (8 inputs), statistics (40) and fewer than ten products and sums.  `size` below is always the sum of the
magnitudes of what is added up, so that cancellation is paid for.  On top comes the rounding to the output's type, half a step of it.
"""
import torch

U = 2.0 ** -24
K = 64
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def rounding(dtype, value):
    """Half a step of the output type at `value`."""
    t = TYPES[dtype]
    info = torch.finfo(t)
    return value.abs() * (info.eps / 2) + info.tiny * info.eps / 2


def norm(v, size, kind, weight, bias, offset, eps):
    """The norm of v's rows, with `size` the magnitudes that v was added up from: (out, error bound of out, standardised, its magnitude, 1/spread)."""
    if kind == "none":
        return v, K * U * size, v, size, None
    if kind == "layer":
        size = size + size.mean(-1, keepdim=True)
        v = v - v.mean(-1, keepdim=True)
    spread = ((v * v).mean(-1, keepdim=True) + eps).sqrt()
    hat, hat_size = v / spread, size / spread
    # an error e of v moves the spread by at most |v . e| / (width spread) <= |e| / sqrt(width), relative to spread
    share = K * U * (hat_size * hat_size).mean(-1, keepdim=True).sqrt()
    error = K * U * hat_size + hat.abs() * (share + K * U)
    out = hat
    if weight is not None:
        out, error = out * (weight + offset), error * (weight.abs() + abs(offset)) + 2 * U * (hat * (weight.abs() + abs(offset))).abs()
    if bias is not None:
        out = out + bias
        error = error + U * (out.abs() + bias.abs())
    return out, error, hat, hat_size, 1 / spread


def gate_of_rows(gate, gate_rows, rows):
    return None if gate is None else torch.repeat_interleave(gate, gate_rows, 0)[:rows]


def forward(parts, residual, gate, gate_rows, p):
    """parts [n_in, rows, width] and the rest in 64 bits; p: settings and parameters by name.  Returns {name: (value, bound without rounding)}."""
    y = parts.sum(0)
    y_size = parts.abs().sum(0)
    n, n_error, _, _, _ = norm(y, y_size, p["post"], p["post_weight"], p["post_bias"], p["weight_offset"], p["post_eps"])
    g = gate_of_rows(gate, gate_rows, y.shape[0])
    factor = p["block_scale"] if g is None else p["block_scale"] * g
    r, r_error = n * factor, n_error * abs(factor) + 3 * U * (n * factor).abs()
    if residual is not None:
        r = r + p["residual_scale"] * residual
        r_error = r_error + 2 * U * (p["residual_scale"] * residual).abs() + U * r.abs()
    h, h_error, _, _, _ = norm(r, r_error / (K * U) + r.abs(), p["pre"], p["pre_weight"], p["pre_bias"], p["weight_offset"], p["pre_eps"])
    return {"folded": (y, 8 * U * y_size), "residual_out": (r, r_error), "outs": (h, h_error)}


def back(d, size, hat, hat_size, rstd, kind):
    """Gradient of a norm's input from d = that of its standardised output; size bounds |d|."""
    along = (d * hat).mean(-1, keepdim=True)
    value = d - hat * along
    total = size + hat_size * (size * hat_size).mean(-1, keepdim=True)
    if kind == "layer":
        value = value - d.mean(-1, keepdim=True)
        total = total + size.mean(-1, keepdim=True)
    return rstd * value, rstd * total


def backward(parts, r, grad_outs, grad_residual_out, gate, gate_rows, p):
    """Gradients in 64 bits from the partial outputs and r as the kernel is given them; {name: (value, bound without rounding)}.
    2 K: statistics come into a gradient twice.  y is folded in 32 bits, with an error that goes by the parts' magnitudes
    (up to 8 u of their sum, however small y itself is), so those are y's size."""
    y = parts.sum(0)
    rows, width = y.shape
    n, _, y_hat, y_size, y_rstd = norm(y, parts.abs().sum(0), p["post"], p["post_weight"], p["post_bias"], p["weight_offset"], p["post_eps"])
    dr, dr_size = grad_residual_out, grad_residual_out.abs()
    found = {}
    depth = 2 * K + rows  # rows are added one after the other at most

    def total(x, size):
        return x.sum(0), depth * U * size.sum(0)

    if grad_outs is not None:
        dh, dh_size = grad_outs.sum(0), grad_outs.abs().sum(0)
        if p["pre"] == "none":
            dr, dr_size = dr + dh, dr_size + dh_size
        else:
            _, _, r_hat, r_size, r_rstd = norm(r, r.abs(), p["pre"], None, None, 0.0, p["pre_eps"])
            w = 1.0 if p["pre_weight"] is None else p["pre_weight"] + p["weight_offset"]
            w_size = 1.0 if p["pre_weight"] is None else p["pre_weight"].abs() + abs(p["weight_offset"])
            d, d_size = back(dh * w, dh_size * w_size, r_hat, r_size, r_rstd, p["pre"])
            dr, dr_size = dr + d, dr_size + d_size
            found["grad_pre_weight"] = total(dh * r_hat, dh_size * r_size)
            found["grad_pre_bias"] = total(dh, dh_size)
    found["grad_residual"] = (p["residual_scale"] * dr, 2 * K * U * abs(p["residual_scale"]) * dr_size)
    c = p["block_scale"]
    g = gate_of_rows(gate, gate_rows, rows)
    w = 1.0 if p["post_weight"] is None else p["post_weight"] + p["weight_offset"]
    w_size = 1.0 if p["post_weight"] is None else p["post_weight"].abs() + abs(p["weight_offset"])
    n_size = y_size * w_size if p["post_bias"] is None else y_size * w_size + p["post_bias"].abs()
    if g is not None:
        groups, pad = gate.shape[0], gate.shape[0] * gate_rows - rows
        each = torch.nn.functional.pad(c * dr * n, (0, 0, 0, pad)).view(groups, gate_rows, width)
        size = torch.nn.functional.pad(abs(c) * dr_size * n_size, (0, 0, 0, pad)).view(groups, gate_rows, width)
        found["grad_gate"] = (each.sum(1), depth * U * size.sum(1))
    factor = c if g is None else c * g
    dn, dn_size = dr * factor, dr_size * abs(factor)
    if p["post"] == "none":
        found["grad_ins"] = (dn, 2 * K * U * dn_size)
    else:
        found["grad_post_weight"] = total(dn * y_hat, dn_size * y_size)
        found["grad_post_bias"] = total(dn, dn_size)
        dy, dy_size = back(dn * w, dn_size * w_size, y_hat, y_size, y_rstd, p["post"])
        found["grad_ins"] = (dy, 4 * K * U * dy_size)
    return found
