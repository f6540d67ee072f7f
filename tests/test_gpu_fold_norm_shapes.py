"""The backward pass of the norms with the calls that have instances of their own: one y and one gradient of h (or none), rows enough
for a team to go through several, at widths around every change of the team's shape; and wide rows of several gradients."""
import pytest

import test_gpu_fold_norm as base

pytestmark = pytest.mark.gpu


def case(types, width, rows, n_in, n_out, kinds, gate_rows, biases, pad, shift, seed):
    return dict(types=types, kinds=kinds, width=width, rows=rows, n_in=n_in, n_out=n_out, gate_rows=gate_rows, weights=True, biases=biases, offset=1.0,
                a=0.75, c=0.5, residual=True, pad=pad, shift=shift, seed=seed)


@pytest.mark.parametrize("biases", [False, True])
@pytest.mark.parametrize("width", [3, 200, 256, 257, 400, 512, 513, 1025, 4095, 4096, 4097, 8191, 8192, 8193, 8704, 9217, 12289, 16379, 16384])
@pytest.mark.parametrize("types", base.TYPES, ids="-".join)
def test_one_gradient(hip, types, width, biases):
    k = base.TYPES.index(types)
    kinds = [("rms", "rms"), ("layer", "rms"), ("rms", "layer"), ("layer", "layer"), ("none", "layer")][(k + width) % 5]
    rows = 1100 if width < 600 else 700 if width < 9000 else 530  # (more than there are teams)
    base.test_backward(hip, case(types, width, rows, 1, 1, kinds, [0, rows // 3, 0, rows][width % 4], biases, width % 3, (width + k) % 9, width + k))


@pytest.mark.parametrize("types", base.TYPES, ids="-".join)
@pytest.mark.parametrize("width,n_in,n_out,gate_rows", [(300, 1, 0, 7), (2000, 1, 0, 0), (9001, 1, 0, 0), (8200, 1, 1, 1), (3000, 1, 1, 2), (8300, 2, 1, 100),
                                                       (10001, 8, 3, 90), (16384, 3, 8, 0), (5000, 6, 5, 0), (700, 4, 2, 33)])
def test_gate_rows_and_several_gradients(hip, types, width, n_in, n_out, gate_rows):
    k = base.TYPES.index(types)
    base.test_backward(hip, case(types, width, 301, n_in, n_out, ("layer", "layer") if k % 2 else ("rms", "layer"), gate_rows, k != 1, k, width % 7, width * 3 + k))
