"""GPU: bits and edges of the 8-bit operators: which roundings a row takes, rows at the ends of f32's range, and results that do not depend on
what shares a call.

Tolerances are those of test_gpu_q8_ops: U = 2^-24 is half a step of f32 relative to the value.
"""
import pytest

import test_gpu_q8_ops as ops8
from test_gpu_q8_ops import U, _check_rows, _dt, _gen, _int8, _norm_error

pytestmark = pytest.mark.gpu


def _at(torch, t, offset):
    """A copy of `t` whose memory starts `offset` elements behind an aligned address."""
    base = torch.empty(t.numel() + offset, dtype=t.dtype, device="cuda")
    base[offset:] = t.flatten()
    return base[offset:].view(t.shape)


def _normed(torch, x, w, eps):
    y = x.double()
    return y / ((y * y).mean(1, keepdim=True) + eps).sqrt() * w.double()


# rows, size, offset of the buffers: one warp and several to a row, groups over resident blocks (odd sizes, many rows), element by element
FORMS = [(3, 64, 0), (300, 2048, 0), (7, 67, 0), (2400, 1024, 0), (4, 40000, 0), (5, 64, 1)]


@pytest.mark.parametrize("rows,size,offset", FORMS)
def test_norm_of_products_next_to_the_smallest(ak, torch_cuda, rows, size, offset):
    """Without eps, h w may be next to 1e-36, from where on a row counts, and y ordinary. A row's largest h w is set just above and below it, and around
    128 times the smallest normal number (1.5e-36)."""
    torch = torch_cuda
    x = 1e-16 * torch.randn(rows, size, device="cuda", generator=_gen(torch, size)).clamp(-2, 2)
    tops = torch.tensor([0.99, 1.01, 1.2, 1.4, 1.5, 1.51, 1.6, 3.0], device="cuda")[torch.arange(rows, device="cuda") % 8]
    x[:, size // 3] = 4e-16
    w = torch.full((size,), 1e-20, device="cuda")
    x *= (tops * 1e-36 / (x[:, size // 3] * w[0]))[:, None]
    x[:, 0] = 0
    x, w = _at(torch, x, offset), _at(torch, w, offset)
    q, scales = torch.full((rows, size), 77, dtype=torch.int8, device="cuda"), torch.full((rows,), 7.0, device="cuda")
    ak.ops.rmsnorm_q8(x, None, w, q, scales, rows, size, 0.0)
    torch.cuda.synchronize()
    none = tops < 1
    assert (q[none] == 0).all() and (scales[none] == 0).all()
    # a product of the smallest kept rows may be subnormal: half a step of these, 2^-150, is 2^-30 of 1e-36 and less
    _check_rows(torch, _normed(torch, x, w, 0.0)[~none], _norm_error(size) + 2.0 ** -30, q[~none], scales[~none])
