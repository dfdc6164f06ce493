"""GPU: the 8-bit operators against their definitions in 64 bits.

Tolerances count roundings. U = 2^-24 is half a step of f32 relative to the value, 2^-8 of bf16, 2^-11 of f16.
"""
import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
HALF = {"f32": 0.0, "bf16": 2.0 ** -8}      # the rounding of the result


def _gen(torch, seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _dt(ak, torch, name):
    return (ak.AK_F32, torch.float32) if name == "f32" else (ak.AK_BF16, torch.bfloat16)


def _int8(torch, shape, g, lo=-127):
    return torch.randint(lo, 128, shape, device="cuda", dtype=torch.int8, generator=g)


# ------------------------------------------------------------------ norm and rows
def _norm_error(size):
    """Relative error of y = h rs w: the squares' sum (a chain of at most 32 in the registers, or size / 512 in the loop, and 10 of the
    reductions), halved by the root; the division, the addition, the root, its reciprocal; two products."""
    return ((max(32, size / 512) + 10) / 2 + 6) * U


def _check_rows(torch, y, tol, q, scales):
    """Rows of int8 against 127 y / max|y|: half a step, and what y and the scale are off."""
    top = y.abs().amax(1)
    assert ((scales.double() - top / 127).abs() <= (2 * tol + 2 * U) * top / 127).all()
    assert q.int().abs().max() <= 127
    assert ((q.double() - 127 * y / top[:, None]).abs() <= 0.5 + 127 * (2 * tol + 3 * U)).all()


@pytest.mark.parametrize("rows,size", [(1, 1), (1, 3), (3, 7), (2, 65), (64, 768), (5, 320), (130, 1001), (297, 64), (300, 2048), (301, 2047), (297, 129), (7, 8192),
                                       (300, 8190), (2, 32765), (2, 32768), (3, 33001), (2, 40000), (2400, 1024), (5003, 1001), (2500, 5001), (700, 14001), (5001, 37)])
@pytest.mark.parametrize("form", ["residual", "plain", "rows", "bf16", "bf16_rows"])
def test_norm(ak, torch_cuda, rows, size, form):
    torch = torch_cuda
    g = _gen(torch, rows + size)
    name = "bf16" if form.startswith("bf16") else "f32"
    dt, tdt = _dt(ak, torch, name)
    x = (3 * torch.randn(rows, size, device="cuda", generator=g)).to(tdt)
    res = torch.randn(rows, size, device="cuda", generator=g) if form == "residual" else None
    w = None if form.endswith("rows") else 1 + 0.2 * torch.randn(size, device="cuda", generator=g)
    pad = torch.full((rows * size + 64,), 99, dtype=torch.int8, device="cuda")
    q, scales = pad[:rows * size].view(rows, size), torch.full((rows,), float("nan"), device="cuda")
    h = x + res if res is not None else x.clone()
    ak.ops.rmsnorm_q8(x, res, w, q, scales, rows, size, 1e-5, in_dtype=dt)
    torch.cuda.synchronize()
    assert torch.equal(x, h)                       # one f32 addition, or nothing
    y, tol = h.double(), 0.0
    if w is not None:
        y = y / ((y * y).mean(1, keepdim=True) + 1e-5).sqrt() * w.double()
        tol = _norm_error(size)
    _check_rows(torch, y, tol, q, scales)
    assert (pad[rows * size:] == 99).all()


@pytest.mark.parametrize("rows,size", [(3, 64), (300, 130)])
def test_norm_at_any_alignment(ak, torch_cuda, rows, size):
    """Buffers that start at an odd element: the same numbers, element by element."""
    torch = torch_cuda
    g = _gen(torch, 5)
    n = rows * size
    base, rbase, w = torch.randn(n + 1, device="cuda", generator=g), torch.randn(n + 3, device="cuda", generator=g), torch.randn(size + 1, device="cuda", generator=g)
    qb = torch.zeros(n + 1, dtype=torch.int8, device="cuda")
    scales = torch.empty(rows, device="cuda")
    h = base[1:].view(rows, size) + rbase[3:].view(rows, size)
    ak.ops.rmsnorm_q8(base[1:], rbase[3:], w[1:], qb[1:], scales, rows, size)
    torch.cuda.synchronize()
    assert torch.equal(base[1:].view(rows, size), h)
    y = h.double()
    y = y / ((y * y).mean(1, keepdim=True) + 1e-5).sqrt() * w[1:].double()
    _check_rows(torch, y, _norm_error(size), qb[1:].view(rows, size), scales)


@pytest.mark.parametrize("size", [64, 65, 2048, 33001])
@pytest.mark.parametrize("norm", [True, False])
def test_rows_without_a_scale(ak, torch_cuda, size, norm):
    """Zeros, values under 1e-30, infinities and NaN: the other rows are as without them."""
    torch = torch_cuda
    x = torch.randn(6, size, device="cuda", generator=_gen(torch, 1))
    x[1] = 0
    x[2] = 1e-31
    x[3, size // 2] = float("nan")
    x[4, size - 1] = -math.inf
    w = torch.ones(size, device="cuda") if norm else None
    q, scales = torch.full((6, size), 77, dtype=torch.int8, device="cuda"), torch.full((6,), 7.0, device="cuda")
    ak.ops.rmsnorm_q8(x, None, w, q, scales, 6, size, 1e-5)
    torch.cuda.synchronize()
    y = x[[0, 5]].double()
    if norm:
        y = y / ((y * y).mean(1, keepdim=True) + 1e-5).sqrt()
    _check_rows(torch, y, _norm_error(size) if norm else 0.0, q[[0, 5]], scales[[0, 5]])
    none = [1, 2, 3, 4]
    if norm:    # row 2 is divided by sqrt(0 + 1e-5): 1e-31 / 3.16e-3 = 3.2e-29 is above 1e-30, a row like any other
        none = [1, 3, 4]
        _check_rows(torch, x[2:3].double() / math.sqrt(1e-5), _norm_error(size), q[2:3], scales[2:3])
    assert (q[none] == 0).all() and (scales[none[:-2]] == 0).all() and scales[3:5].isnan().all()


@pytest.mark.parametrize("size", [4000, 4001])
def test_norm_of_more_than_32_bits_of_values(ak, torch_cuda, size):
    torch = torch_cuda
    rows, n = 1100000, 5
    x = torch.zeros(rows, size, dtype=torch.bfloat16, device="cuda")
    x[-n:] = torch.randn(n, size, device="cuda", generator=_gen(torch, 1)).bfloat16()
    w = 1 + 0.2 * torch.randn(size, device="cuda", generator=_gen(torch, 2))
    q, scales = torch.full((rows, size), 77, dtype=torch.int8, device="cuda"), torch.full((rows,), 7.0, device="cuda")
    ak.ops.rmsnorm_q8(x, None, w, q, scales, rows, size, in_dtype=ak.AK_BF16)
    torch.cuda.synchronize()
    y = x[-n:].double()
    _check_rows(torch, y / ((y * y).mean(1, keepdim=True) + 1e-5).sqrt() * w.double(), _norm_error(size), q[-n:], scales[-n:])
    assert (scales[:-n] == 0).all() and not q[rows - n - 3:rows - n].any()


@pytest.mark.parametrize("rows,size", [(2500, 1001), (2400, 2048), (9, 1003), (300, 64)])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_rows_between_rows_without_a_scale(ak, torch_cuda, rows, size, dtype):
    """Every third row holds NaN or infinities only: nothing of it reaches its neighbours, which share 16-byte words with it in odd sizes."""
    torch = torch_cuda
    dt, tdt = _dt(ak, torch, dtype)
    x = torch.randn(rows, size, device="cuda", generator=_gen(torch, rows)).to(tdt)
    x[1::3] = float("nan")
    x[4::6] = math.inf
    w = 1 + 0.2 * torch.randn(size, device="cuda", generator=_gen(torch, 3))
    q, scales = torch.full((rows, size), 77, dtype=torch.int8, device="cuda"), torch.full((rows,), 7.0, device="cuda")
    ak.ops.rmsnorm_q8(x, None, w, q, scales, rows, size, 1e-5, in_dtype=dt)
    torch.cuda.synchronize()
    assert (q[1::3] == 0).all() and scales[1::3].isnan().all()
    keep = torch.arange(rows, device="cuda") % 3 != 1
    y = x[keep].double()
    _check_rows(torch, y / ((y * y).mean(1, keepdim=True) + 1e-5).sqrt() * w.double(), _norm_error(size), q[keep], scales[keep])


@pytest.mark.parametrize("size", [64, 67])
def test_norm_of_small_products(ak, torch_cuda, size):
    """Without eps a row may be tiny and y ordinary. h w of 1e-35 is a row like any other, under 1e-36 it counts as zero."""
    torch = torch_cuda
    x = torch.randn(2, size, device="cuda", generator=_gen(torch, 1)).clamp(-3, 3)
    x[0] *= 1e-15
    x[1] *= 1e-18
    w = torch.full((size,), 1e-20, device="cuda")
    q, scales = torch.full((2, size), 77, dtype=torch.int8, device="cuda"), torch.full((2,), 7.0, device="cuda")
    ak.ops.rmsnorm_q8(x, None, w, q, scales, 2, size, 0.0)
    torch.cuda.synchronize()
    y = x[:1].double()
    _check_rows(torch, y / (y * y).mean(1, keepdim=True).sqrt() * w.double(), _norm_error(size), q[:1], scales[:1])
    assert (q[1] == 0).all() and scales[1] == 0


# ------------------------------------------------------------------ product
def _gemm(ak, torch, m, n, k, epi, pad=0, seed=0, lo=-127):
    g = _gen(torch, seed + m * 7 + n * 3 + k)
    a, wt = _int8(torch, (m, k), g, lo), _int8(torch, (n, k), g, lo)
    sa, sw = 0.01 + torch.rand(m, device="cuda", generator=g), (0.01 + torch.rand(n, device="cuda", generator=g)) / k
    ld = n + pad
    c = torch.full((m + 1, ld), 3.25, device="cuda", dtype=torch.float32 if epi < 2 else torch.bfloat16)
    if epi == 1:
        c[:m, :n] = torch.randn(m, n, device="cuda", generator=g)
    c0 = c.clone()
    ak.ops.gemm_q8(a, sa, wt, sw, c, m, n, k, epi, ldc=ld if pad else 0)
    torch.cuda.synchronize()
    v = (a.double() @ wt.double().t()) * sa.double()[:, None] * sw.double()      # sums below 2^53: exact
    got = c[:m, :n].double()
    if epi == 0:
        want, tol = v, 3 * U * v.abs()               # the sum to f32, two products
    elif epi == 1:
        want = v + c0[:m, :n].double()
        tol = 3 * U * v.abs() + U * want.abs() * (1 + 4 * U)
    elif epi == 2:
        want, tol = v, (2.0 ** -8 + 4 * U) * v.abs()
    else:
        want = v * torch.sigmoid(v)
        tol = (2.0 ** -8 + 2.0 ** -16) * want.abs() + 1e-35   # the activation to 2^-17 of its value (and 0 where it is below 2e-36)
    bad = (got - want).abs() > tol
    assert not bad.any(), (int(bad.sum()), float(((got - want).abs() / want.abs().clamp(min=1e-30)).max()))
    assert torch.equal(c[m], c0[m]) and (pad == 0 or torch.equal(c[:m, n:], c0[:m, n:]))   # behind the rows and the columns


@pytest.mark.parametrize("epi", [0, 1, 2, 3])
@pytest.mark.parametrize("m,n,k,pad", [(1, 1, 16, 0), (1, 16, 16, 0), (1, 33, 128, 3), (2, 2304, 768, 0), (16, 960, 320, 0), (17, 1001, 144, 7), (33, 50, 8192, 2),
                                       (63, 257, 4096, 0), (64, 6144, 2048, 0), (65, 320, 1280, 0), (100, 8192, 2048, 0), (128, 768, 2080, 0), (129, 48, 272, 0),
                                       (200, 2304, 768, 1), (1000, 777, 400, 0), (1023, 2048, 1024, 0), (3, 50257, 320, 7), (2, 50257, 64, 0)])
def test_gemm(ak, torch_cuda, epi, m, n, k, pad):
    _gemm(ak, torch_cuda, m, n, k, epi, pad)


@pytest.mark.parametrize("epi", [0, 1, 2, 3])
@pytest.mark.parametrize("m,n,k,pad", [(1024, 256, 16, 0), (1025, 257, 400, 0), (1500, 300, 2048, 4), (2049, 2304, 768, 0), (1200, 1003, 144, 5), (5000, 511, 128, 1)])
def test_gemm_of_many_rows(ak, torch_cuda, epi, m, n, k, pad):
    _gemm(ak, torch_cuda, m, n, k, epi, pad)


@pytest.mark.parametrize("n", [65600, 65601])
def test_gemm_of_more_than_32_bits_of_results(ak, torch_cuda, n):
    torch = torch_cuda
    m, k, last = 70001, 32, 130
    g = _gen(torch, n)
    a, wt = _int8(torch, (m, k), g), _int8(torch, (n, k), g)
    sa, sw = 0.01 + torch.rand(m, device="cuda", generator=g), (0.01 + torch.rand(n, device="cuda", generator=g)) / k
    c = torch.full((m, n), 3.25, dtype=torch.bfloat16, device="cuda")
    ak.ops.gemm_q8(a, sa, wt, sw, c, m, n, k, ak.EPI_STORE_BF16)
    torch.cuda.synchronize()
    want = (a[-last:].double() @ wt.double().t()) * sa[-last:].double()[:, None] * sw.double()
    assert ((c[-last:].double() - want).abs() <= (2.0 ** -8 + 4 * U) * want.abs()).all()


@pytest.mark.parametrize("m,n", [(1, 40), (130, 64), (1024, 256)])
def test_gemm_sums_at_their_limits(ak, torch_cuda, m, n):
    """-128 everywhere over the longest K (2^31 less 2^18), and the odd sums next to it."""
    torch = torch_cuda
    k = 131056
    a = torch.full((m, k), -128, dtype=torch.int8, device="cuda")
    wt = torch.full((n, k), -128, dtype=torch.int8, device="cuda")
    wt[n // 2] = 127
    a[0, 5] = -127
    one_m, one_n = torch.ones(m, device="cuda"), torch.ones(n, device="cuda")
    c = torch.empty(m, n, device="cuda")
    ak.ops.gemm_q8(a, one_m, wt, one_n, c, m, n, k)
    torch.cuda.synchronize()
    want = torch.full((m, n), 16384 * k, dtype=torch.float64, device="cuda")
    want[:, n // 2] = -128 * 127 * k
    want[0] -= torch.where(torch.arange(n, device="cuda") == n // 2, -127.0, 128.0).double()
    assert torch.equal(c.double(), want.float().double())


def test_gemm_rows_do_not_depend_on_the_batch(ak, torch_cuda):
    """One row, a decode batch, a prompt: the same bits, whatever kernel and split they ran on."""
    torch = torch_cuda
    g = _gen(torch, 3)
    n, k = 768, 2304
    a, wt = _int8(torch, (2048, k), g), _int8(torch, (n, k), g)
    sa, sw = torch.rand(2048, device="cuda", generator=g), torch.rand(n, device="cuda", generator=g)
    full = torch.empty(2048, n, device="cuda")
    ak.ops.gemm_q8(a, sa, wt, sw, full, 2048, n, k)
    for m in (1, 8, 64, 128, 500):
        c = torch.empty(m, n, device="cuda")
        ak.ops.gemm_q8(a[:m], sa[:m], wt, sw, c, m, n, k)
        torch.cuda.synchronize()
        assert torch.equal(c, full[:m]), m


@pytest.mark.parametrize("m,n,k", [(5, 100, 64), (64, 2048, 4096), (1300, 520, 256)])
def test_gemm_scales_at_any_alignment(ak, torch_cuda, m, n, k):
    """Scales that begin at an odd element: the same bits."""
    torch = torch_cuda
    g = _gen(torch, 6)
    a, wt = _int8(torch, (m, k), g), _int8(torch, (n, k), g)
    sa, sw = torch.rand(m + 1, device="cuda", generator=g), torch.rand(n + 1, device="cuda", generator=g)
    c, want = torch.empty(m, n, device="cuda"), torch.empty(m, n, device="cuda")
    ak.ops.gemm_q8(a, sa[1:], wt, sw[1:], c, m, n, k)
    ak.ops.gemm_q8(a, sa[1:].clone(), wt, sw[1:].clone(), want, m, n, k)
    torch.cuda.synchronize()
    assert torch.equal(c, want)


@pytest.mark.parametrize("m", [3, 1100])
def test_gemm_passes_scales_that_are_not_finite_on(ak, torch_cuda, m):
    torch = torch_cuda
    g = _gen(torch, 3)
    n, k = 300, 256
    a, wt = _int8(torch, (m, k), g), _int8(torch, (n, k), g)
    sa, sw = torch.ones(m, device="cuda"), torch.ones(n, device="cuda")
    sa[1], sw[7], a[1] = float("nan"), float("nan"), 0
    c = torch.empty(m, n, device="cuda")
    ak.ops.gemm_q8(a, sa, wt, sw, c, m, n, k)
    torch.cuda.synchronize()
    want = a.double() @ wt.double().t()
    want[1], want[:, 7] = float("nan"), float("nan")
    assert torch.equal(c.double().nan_to_num(1e30), want.nan_to_num(1e30))    # sums below 2^24: exact in f32


# ------------------------------------------------------------------ cache
def _cache(torch, blocks, kv_heads, hd, seed):
    g = _gen(torch, seed)
    kp, vp = _int8(torch, (blocks, kv_heads, 16, hd), g), _int8(torch, (blocks, kv_heads, 16, hd), g)
    ks, vs = (0.002 + 0.03 * torch.rand(blocks, kv_heads, 16, device="cuda", generator=g) for _ in range(2))
    return kp, vp, ks, vs


def _rope_table(torch, n, hd):
    inv = 10000.0 ** (-torch.arange(0, hd, 2, dtype=torch.float64, device="cuda") / hd)
    a = torch.arange(n, dtype=torch.float64, device="cuda")[:, None] * inv
    return torch.stack([a.cos(), a.sin()], -1).float().contiguous()


def _turn(x, cs):
    """x [tokens, heads, hd] in 64 bits; cs [tokens, hd / 2, 2]. And the size of the terms, for the roundings."""
    import torch
    a, b, c, s = x[..., 0::2], x[..., 1::2], cs[:, None, :, 0], cs[:, None, :, 1]
    y = torch.stack([a * c - b * s, a * s + b * c], -1).flatten(-2)
    size = torch.stack([(a * c).abs() + (b * s).abs(), (a * s).abs() + (b * c).abs()], -1).flatten(-2)
    return y, size


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("tokens,heads,kv_heads,hd", [(1, 1, 1, 32), (1, 5, 5, 64), (7, 6, 3, 96), (64, 12, 12, 64), (33, 16, 2, 128), (3, 8, 1, 128), (130, 4, 4, 32),
                                                      (1000, 12, 4, 96)])
def test_append(ak, torch_cuda, dtype, tokens, heads, kv_heads, hd):
    torch = torch_cuda
    dt, tdt = _dt(ak, torch, dtype)
    g = _gen(torch, tokens + hd)
    blocks = tokens // 16 + 3
    x = torch.randn(tokens, heads + 2 * kv_heads, hd, device="cuda", generator=g)
    table = _rope_table(torch, 700, hd)
    pos = torch.randint(0, 700, (tokens,), device="cuda", generator=g, dtype=torch.int32)
    slots = torch.randperm(blocks * 16, device="cuda", generator=g)[:tokens].to(torch.int32)
    kp, vp, ks, vs = _cache(torch, blocks, kv_heads, hd, 1)
    before = [t.clone() for t in (kp, vp, ks, vs)]
    q = torch.full((tokens, heads * hd), 9.0, device="cuda", dtype=tdt)
    off, unslotted = [], []
    if tokens > 6:      # left out by their position, and by their slot
        pos[2], pos[3] = 700, -1
        slots[4], slots[5] = -1, blocks * 16
        off, unslotted = [2, 3], [4, 5]
    ak.ops.rope_kv_append_q8(x, table, 700, pos, slots, q, kp, vp, ks, vs, tokens, heads, kv_heads, hd, blocks, dtype=dt)
    torch.cuda.synchronize()
    live = torch.tensor([t for t in range(tokens) if t not in off], device="cuda")
    kept = torch.tensor([t for t in range(tokens) if t not in off + unslotted], device="cuda")
    y, size = _turn(x[:, :heads + kv_heads].double(), table[pos.clamp(0, 699).long()].double())
    got = q.view(tokens, heads, hd).double()
    assert ((got - y[:, :heads]).abs() <= HALF[dtype] * (1 + 4 * U) * y[:, :heads].abs() + 2 * U * size[:, :heads])[live].all()   # two products, one sum
    assert all((got[t] == 9).all() for t in off)
    s = slots[kept].long()
    block, place = s // 16, s % 16
    for pool, scales, want, terms in ((kp, ks, y[:, heads:], size[:, heads:]), (vp, vs, x[:, heads + kv_heads:].double(), None)):
        want, err = want[kept].flatten(0, 1), 0.0
        if terms is not None:   # relative to the row's largest value: a term is at most sqrt(2) of it
            err = 2 * U * float((terms[kept].flatten(0, 1).amax(1) / want.abs().amax(1)).max())
        _check_rows(torch, want, err, pool[block, :, place].flatten(0, 1), scales[block, :, place].flatten())
    for now, was in zip((kp, vp, ks, vs), before):      # every other slot
        now, was = now.clone(), was.clone()
        now[block, :, place] = 0
        was[block, :, place] = 0
        assert torch.equal(now, was)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("tokens,kv_heads,hd", [(1, 1, 32), (5, 3, 96), (64, 12, 64), (1000, 8, 128), (17, 5, 64)])
def test_read(ak, torch_cuda, dtype, tokens, kv_heads, hd):
    torch = torch_cuda
    dt, tdt = _dt(ak, torch, dtype)
    blocks = 7
    kp, vp, ks, vs = _cache(torch, blocks, kv_heads, hd, 2)
    slots = torch.randint(0, blocks * 16, (tokens,), device="cuda", generator=_gen(torch, 4), dtype=torch.int32)    # repeated ones among them
    if tokens > 4:
        slots[1], slots[3] = -1, blocks * 16
    have = (slots >= 0) & (slots < blocks * 16)
    s = slots.clamp(0, blocks * 16 - 1).long()
    k_out, v_out = (torch.full((tokens, kv_heads * hd), 5.0, device="cuda", dtype=tdt) for _ in range(2))
    ak.ops.kv_read_q8(kp, vp, ks, vs, slots, k_out, v_out, tokens, kv_heads, hd, blocks, dtype=dt)
    torch.cuda.synchronize()
    for pool, scales, out in ((kp, ks, k_out), (vp, vs, v_out)):
        want = (pool[s // 16, :, s % 16].float() * scales[s // 16, :, s % 16][..., None]).flatten(1)
        want = torch.where(have[:, None], want, torch.zeros_like(want)).to(tdt)
        assert torch.equal(out, want)
    one = torch.full_like(k_out, 5.0)
    ak.ops.kv_read_q8(kp, vp, ks, vs, slots, None, one, tokens, kv_heads, hd, blocks, dtype=dt)
    torch.cuda.synchronize()
    assert torch.equal(one, v_out)


# ------------------------------------------------------------------ attention
def _attn_case(torch, lens, kv_heads, hd, seed, spare=3):
    """A cache with sequences of `lens` in random blocks; unused positions and blocks hold garbage, NaN for scales included."""
    per = [-(-n // 16) for n in lens]
    blocks = sum(per) + spare
    kp, vp, ks, vs = _cache(torch, blocks, kv_heads, hd, seed)
    order = torch.randperm(blocks, device="cuda", generator=_gen(torch, seed)).to(torch.int32)
    max_blocks = max(max(per), 1) + 1
    tables = torch.full((len(lens), max_blocks), 1 << 30, dtype=torch.int32, device="cuda")
    at = 0
    used = torch.zeros(blocks, 16, dtype=torch.bool, device="cuda")
    for r, (n, p) in enumerate(zip(lens, per)):
        tables[r, :p] = order[at:at + p]
        pos = torch.arange(n, device="cuda")
        used[tables[r].long()[pos // 16], pos % 16] = True
        at += p
    ks.masked_fill_(~used[:, None], float("nan"))
    vs.masked_fill_(~used[:, None], float("nan"))
    return (kp, vp, ks, vs), tables, torch.tensor(lens, dtype=torch.int32, device="cuda"), blocks, max_blocks


def _attn_check(torch, out, q, cache, tables, lens, q_len, heads, kv_heads, hd, scale, dtype, blocks, splits=16):
    kp, vp, ks, vs = (t.double() for t in cache)
    group = heads // kv_heads
    out, q = out.double().view(len(lens), q_len, kv_heads, group, hd), q.double().view(len(lens), q_len, kv_heads, group, hd)
    rounded = dtype == "bf16" and q_len * group > 4      # weights rounded to f16
    for r, n in enumerate(lens):
        ids = tables[r].long()
        pos = torch.arange(min(max(n, 0), tables.shape[1] * 16), device="cuda")
        b = ids[pos // 16]
        pos, b = pos[(b >= 0) & (b < blocks)], b[(b >= 0) & (b < blocks)]
        for i in range(q_len):
            see = pos <= n - q_len + i
            p, bb = pos[see], b[see]
            if not len(p):
                assert (out[r, i] == 0).all()
                continue
            k, v = kp[bb, :, p % 16] * ks[bb, :, p % 16][..., None], vp[bb, :, p % 16] * vs[bb, :, p % 16][..., None]
            s = torch.einsum("kgd,jkd->kgj", q[r, i], k) * scale
            size = torch.einsum("kgd,jkd->kgj", q[r, i].abs(), k.abs()) * abs(scale)
            w = torch.softmax(s, -1)
            want, mass = torch.einsum("kgj,jkd->kgd", w, v), torch.einsum("kgj,jkd->kgd", w, v.abs())
            # A score: HD / 16 steps of a sum and the scales, each off by at most 2^-22 of the terms, and what the query is off. A weight: that
            # (and the maximum's, alike), exp2 and the exponent's rounding. The sums: a step of the tensor core per 16 positions.
            # Queries are integers of D base-256 digits, half a step of 127 * 256^(D - 1) of the head's largest value.
            digits = q[r, i].abs().amax(-1, keepdim=True) * 2.0 ** (-24 if dtype == "f32" else -16)
            size = size * (hd / 16 + 6) * 2.0 ** -22 + torch.einsum("kgd,jkd->kgj", digits.expand(q[r, i].shape), k.abs()) * abs(scale)
            ds = float(size.max())
            rel = 2 * (ds + 2.0 ** -21) + (len(p) / 16 + 40) * 2.0 ** -22 + (2.0 ** -11 if rounded else 0)
            tol = rel * mass + HALF[dtype] * want.abs()
            err = (out[r, i] - want).abs()
            assert (err <= tol).all(), (r, i, n, float((err / tol).max()), float(err.max()))


def _attn(ak, torch, lens, q_len, heads, kv_heads, hd, dtype, n_splits=0, seed=0, scale=None, q_size=2.0):
    dt, tdt = _dt(ak, torch, dtype)
    scale = hd ** -0.5 if scale is None else scale
    cache, tables, klens, blocks, mb = _attn_case(torch, lens, kv_heads, hd, seed)
    q = (q_size * torch.randn(len(lens) * q_len, heads * hd, device="cuda", generator=_gen(torch, seed + 1))).to(tdt)
    out = torch.full_like(q, 7.0)
    ak.ops.attn_decode_paged_q8(q, *cache, tables, klens, out, len(lens), q_len, heads, kv_heads, hd, mb, scale, blocks, dtype=dt, n_splits=n_splits)
    torch.cuda.synchronize()
    _attn_check(torch, out, q, cache, tables, lens, q_len, heads, kv_heads, hd, scale, dtype, blocks)
    return out


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("hd", [32, 64, 96, 128])
@pytest.mark.parametrize("heads,kv_heads", [(3, 3), (8, 2), (5, 1), (16, 1)])
def test_attn_decode(ak, torch_cuda, dtype, hd, heads, kv_heads):
    _attn(ak, torch_cuda, [0, 1, 2, 15, 16, 17, 64, 65, 301, 1000], 1, heads, kv_heads, hd, dtype)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("q_len,heads,kv_heads,hd", [(2, 4, 4, 64), (4, 8, 2, 128), (5, 2, 2, 32), (3, 6, 2, 96), (9, 2, 2, 64), (17, 4, 2, 128), (40, 1, 1, 64)])
def test_attn_of_several_new_tokens(ak, torch_cuda, dtype, q_len, heads, kv_heads, hd):
    """Drafted tokens and chunks of prompts, sequences shorter than the chunk among them."""
    _attn(ak, torch_cuda, [0, 1, 3, 16, 17, 33, 200, 513], q_len, heads, kv_heads, hd, dtype)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("n_splits", [1, 2, 3, 4, 5, 7, 8, 11, 13, 16])
def test_attn_splits(ak, torch_cuda, dtype, n_splits):
    """Any number of splits, most of them empty for the short sequences."""
    _attn(ak, torch_cuda, [0, 1, 40, 700, 3001], 2, 6, 3, 64, dtype, n_splits)
    _attn(ak, torch_cuda, [5, 129, 2000], 1, 8, 1, 128, dtype, n_splits)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_attn_long(ak, torch_cuda, dtype):
    _attn(ak, torch_cuda, [40000], 1, 2, 2, 64, dtype)
    _attn(ak, torch_cuda, [30011, 9], 4, 8, 2, 128, dtype)
    _attn(ak, torch_cuda, [4000, 2001, 17], 1, 12, 12, 64, dtype)
    _attn(ak, torch_cuda, [6000] * 5, 1, 10, 5, 96, dtype)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("q_size,scale", [(1e-20, 1e20), (1e20, 1e-21), (30.0, 0.1), (1.0, 0.0), (1.0, -0.125)])
def test_attn_ranges(ak, torch_cuda, dtype, q_size, scale):
    """Queries far outside f16's range, peaked scores, equal and reversed ones."""
    _attn(ak, torch_cuda, [1, 100, 515], 1, 4, 2, 64, dtype, q_size=q_size, scale=scale)


def test_attn_value_scales_of_all_sizes(ak, torch_cuda):
    """Value scales over 12 orders of magnitude, growing and shrinking along a sequence."""
    torch = torch_cuda
    lens, hd = [600, 600], 64
    cache, tables, klens, blocks, mb = _attn_case(torch, lens, 2, hd, 9)
    for r in range(2):
        for j in range(38):
            cache[3][tables[r, j].long()] *= 10.0 ** ((j if r == 0 else 37 - j) / 37 * 12 - 6)
    q = 0.2 * torch.randn(2, 4 * hd, device="cuda", generator=_gen(torch, 1))
    out = torch.empty_like(q)
    for n_splits in (1, 4):
        ak.ops.attn_decode_paged_q8(q, *cache, tables, klens, out, 2, 1, 4, 2, hd, mb, 0.125, blocks, dtype=ak.AK_F32, n_splits=n_splits)
        torch.cuda.synchronize()
        _attn_check(torch, out, q, cache, tables, lens, 1, 4, 2, hd, 0.125, "f32", blocks)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("n_splits", [1, 2])
def test_attn_large_value_that_no_query_looks_at(ak, torch_cuda, dtype, n_splits):
    """A value a million times the others at a position whose weight vanishes."""
    torch = torch_cuda
    dt, tdt = _dt(ak, torch, dtype)
    lens, heads, hd = [40, 300], 3, 64
    cache, tables, klens, blocks, mb = _attn_case(torch, lens, heads, hd, 5)
    q = torch.randn(2, heads * hd, device="cuda", generator=_gen(torch, 2)).to(tdt)
    big = 2.0 ** 20 * float(cache[3].nan_to_num(0.0).max())
    for r in range(2):
        b, p = int(tables[r, 1]), 3
        cache[0][b, :, p] = (-127 * q[r].view(heads, hd).float().sign()).to(torch.int8)
        cache[2][b, :, p] = 1.0      # scores of -127 * sum |q| / 8, some -800
        cache[3][b, :, p] = big
    out = torch.empty_like(q)
    ak.ops.attn_decode_paged_q8(q, *cache, tables, klens, out, 2, 1, heads, heads, hd, mb, 0.125, blocks, dtype=dt, n_splits=n_splits)
    torch.cuda.synchronize()
    kp, vp, ks, vs = (t.double() for t in cache)
    for r, n in enumerate(lens):
        pos = torch.arange(n, device="cuda")
        b, p = tables[r].long()[pos // 16], pos % 16
        k, v, x = kp[b, :, p] * ks[b, :, p][..., None], vp[b, :, p] * vs[b, :, p][..., None], q[r].view(heads, hd).double()
        w = torch.softmax(torch.einsum("kd,jkd->kj", x, k) * 0.125, -1)
        want, mass = torch.einsum("kj,jkd->kd", w, v), torch.einsum("kj,jkd->kd", w, v.abs())
        # As in _attn_check, of the positions that weigh anything; and for every position half a step of f16's smallest numbers, 2^-25 / 2^11 with the
        # factor of a weight's rest, in units of at most 2 * 2^-5 of the largest value scale.
        k = k[pos != 19].abs()
        size = torch.einsum("kd,jkd->kj", x.abs(), k) * (hd / 16 + 6) * 2.0 ** -22
        size = 0.125 * (size + x.abs().amax(-1)[:, None] * k.sum(-1).T * 2.0 ** (-24 if dtype == "f32" else -16))
        rel = 2 * (float(size.max()) + 2.0 ** -21) + (n / 16 + 40) * 2.0 ** -22
        err = (out[r].view(heads, hd).double() - want).abs()
        tol = rel * mass + HALF[dtype] * want.abs() + n * 2.0 ** -40 * 127 * big
        assert (err <= tol).all(), (r, float((err / tol).max()))


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("q_len", [1, 5])
def test_attn_blocks_outside_the_pool(ak, torch_cuda, dtype, q_len):
    """Their positions are left out, whole sequences of them give zeros; lengths past the table are cut."""
    torch = torch_cuda
    dt, tdt = _dt(ak, torch, dtype)
    lens, hd = [300, 70, 64, 500], 64
    cache, tables, klens, blocks, mb = _attn_case(torch, lens, 2, hd, 3)
    for t in cache[2:]:
        t.nan_to_num_(0.01)
    tables[0, 3], tables[0, 18], tables[0, 0] = -1, blocks, -(1 << 31)
    tables[2] = -1
    lens = [300, 70, 64, mb * 16 + 900]     # the last one's table has entries for mb * 16 positions, the last of them outside the pool
    klens = torch.tensor(lens, dtype=torch.int32, device="cuda")
    q = torch.randn(4 * q_len, 4 * hd, device="cuda", generator=_gen(torch, 1)).to(tdt)
    out = torch.full_like(q, 7.0)
    ak.ops.attn_decode_paged_q8(q, *cache, tables, klens, out, 4, q_len, 4, 2, hd, mb, 0.125, blocks, dtype=dt)
    torch.cuda.synchronize()
    _attn_check(torch, out, q, cache, tables, lens, q_len, 4, 2, hd, 0.125, dtype, blocks)


def test_attn_values_that_are_not_finite(ak, torch_cuda):
    """A NaN in a query or in a scale that a query sees is that query's result, and no other's."""
    torch = torch_cuda
    lens, hd = [100, 100, 100], 64
    cache, tables, klens, blocks, mb = _attn_case(torch, lens, 2, hd, 3)
    q = torch.randn(6, 4 * hd, device="cuda", generator=_gen(torch, 1))
    q[2, 70] = float("inf")                                   # sequence 1, its first query, head 1
    cache[2][tables[2, 6].long(), 1, 3] = float("nan")        # sequence 2, position 99 (the newest), kv head 1
    out = torch.zeros_like(q)
    ak.ops.attn_decode_paged_q8(q, *cache, tables, klens, out, 3, 2, 4, 2, hd, mb, 0.125, blocks, dtype=ak.AK_F32)
    torch.cuda.synchronize()
    bad = out.view(3, 2, 4, hd).isnan()
    want = torch.zeros(3, 2, 4, dtype=torch.bool, device="cuda")
    want[1, 0, 1], want[2, 1, 2:] = True, True                # the first query does not see position 99
    assert torch.equal(bad.all(-1), want) and torch.equal(bad.any(-1), want)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("hd,q_len,heads", [(32, 1, 4), (64, 1, 2), (64, 3, 8), (96, 1, 2), (96, 5, 4), (128, 1, 2), (128, 2, 8)])
def test_attn_bits_do_not_depend_on_what_nobody_sees(ak, torch_cuda, dtype, hd, q_len, heads):
    """Behind a sequence's end, in the rest of its last block, lies anything: the same bits come out."""
    torch = torch_cuda
    dt, tdt = _dt(ak, torch, dtype)
    lens = [500, 37, 1000, 1, 15, 333, 90, 2001, 700, 701, 702, 703, 1234, 60]
    cache, tables, klens, blocks, mb = _attn_case(torch, lens, 2, hd, 3)
    unseen = cache[2].isnan()
    q = (2 * torch.randn(len(lens) * q_len, heads * hd, device="cuda", generator=_gen(torch, 1))).to(tdt)
    outs = []
    for k_scale, v_scale in ((float("nan"), float("nan")), (1e-3, 1e25), (1e3, 1e-25)):
        cache[2].masked_fill_(unseen, k_scale)
        cache[3].masked_fill_(unseen, v_scale)
        out = torch.empty_like(q)
        ak.ops.attn_decode_paged_q8(q, *cache, tables, klens, out, len(lens), q_len, heads, 2, hd, mb, hd ** -0.5, blocks, dtype=dt)
        outs.append(out)
    torch.cuda.synchronize()
    assert torch.equal(outs[0], outs[1]) and torch.equal(outs[0], outs[2])


def test_attn_far_blocks(ak, torch_cuda):
    """Offsets past 32 bits: pools of 4.3 GB each, the sequences at their ends."""
    torch = torch_cuda
    kv_heads, hd, blocks = 16, 128, 131200
    kp, vp = (torch.empty(blocks, kv_heads, 16, hd, dtype=torch.int8, device="cuda") for _ in range(2))
    ks, vs = (torch.empty(blocks, kv_heads, 16, device="cuda") for _ in range(2))
    small, tables, klens, few, mb = _attn_case(torch, [90, 33], kv_heads, hd, 4)
    for t, s in zip((kp, vp, ks, vs), small):
        t[blocks - few:] = s
    tables += blocks - few
    x = torch.randn(1, 3 * kv_heads, hd, device="cuda", generator=_gen(torch, 2))
    slot = torch.tensor([int(tables[0, 5]) * 16 + 9], dtype=torch.int32, device="cuda")     # position 89
    q, back = torch.empty(1, kv_heads * hd, device="cuda"), torch.empty(1, kv_heads * hd, device="cuda")
    ak.ops.rope_kv_append_q8(x, _rope_table(torch, 100, hd), 100, torch.tensor([89], dtype=torch.int32, device="cuda"), slot, q, kp, vp, ks, vs, 1, kv_heads,
                             kv_heads, hd, blocks, dtype=ak.AK_F32)
    ak.ops.kv_read_q8(kp, vp, ks, vs, slot, None, back, 1, kv_heads, hd, blocks, dtype=ak.AK_F32)
    v = x[0, 2 * kv_heads:]
    assert ((back.view(kv_heads, hd) - v).abs() <= (0.5 + 1e-4) / 127 * v.abs().amax(1, keepdim=True)).all()
    qq = torch.randn(2, kv_heads * hd, device="cuda", generator=_gen(torch, 3))
    out = torch.empty_like(qq)
    ak.ops.attn_decode_paged_q8(qq, kp, vp, ks, vs, tables, klens, out, 2, 1, kv_heads, kv_heads, hd, mb, 0.1, blocks, dtype=ak.AK_F32)
    torch.cuda.synchronize()
    end = tuple(t[blocks - few:].clone() for t in (kp, vp, ks, vs))
    _attn_check(torch, out, qq, end, tables - (blocks - few), [90, 33], 1, kv_heads, kv_heads, hd, 0.1, "f32", few)


# ------------------------------------------------------------------ streams, graphs
def _work(ak, torch, seed):
    """One call of every operator on buffers of its own: (call(stream), the outputs). Odd seeds: a decode step of 40 sequences; even ones: long
    sequences that are split, and a product of many rows."""
    g = _gen(torch, seed)
    if seed % 2 == 0:
        x, w = torch.randn(2048, 768, device="cuda", generator=g), torch.rand(768, device="cuda", generator=g)
        q8, s8 = torch.empty(2048, 768, dtype=torch.int8, device="cuda"), torch.empty(2048, device="cuda")
        wt, sw = _int8(torch, (1536, 768), g), torch.rand(1536, device="cuda", generator=g)
        y, out = torch.empty(2048, 1536, device="cuda"), torch.empty(2, 768, device="cuda")
        cache, tables, klens, blocks, mb = _attn_case(torch, [5000, 4099], 12, 64, seed)

        def long_call(stream):
            ak.ops.rmsnorm_q8(x, None, w, q8, s8, 2048, 768, stream=stream)
            ak.ops.gemm_q8(q8, s8, wt, sw, y, 2048, 1536, 768, stream=stream)
            ak.ops.attn_decode_paged_q8(x, *cache, tables, klens, out, 2, 1, 12, 12, 64, mb, 0.125, blocks, dtype=ak.AK_F32, stream=stream)
        return long_call, [q8, s8, y, out], x
    x, w = torch.randn(40, 768, device="cuda", generator=g), torch.rand(768, device="cuda", generator=g)
    q8, s8 = torch.empty(40, 768, dtype=torch.int8, device="cuda"), torch.empty(40, device="cuda")
    wt, sw = _int8(torch, (2304, 768), g), torch.rand(2304, device="cuda", generator=g)
    qkv = torch.empty(40, 2304, device="cuda")
    cache, tables, klens, blocks, mb = _attn_case(torch, [400] * 40, 12, 64, seed)
    for t in cache[2:]:
        t.nan_to_num_(0.01)
    pos = klens - 1
    slots = (tables[:, 399 // 16] * 16 + 399 % 16).int()
    q, out = torch.empty(40, 768, device="cuda", dtype=torch.bfloat16), torch.empty(40, 768, device="cuda", dtype=torch.bfloat16)
    k_out, v_out = torch.empty(40, 768, device="cuda"), torch.empty(40, 768, device="cuda")
    table = _rope_table(torch, 512, 64)

    def call(stream):
        ak.ops.rmsnorm_q8(x, None, w, q8, s8, 40, 768, stream=stream)
        ak.ops.gemm_q8(q8, s8, wt, sw, qkv, 40, 2304, 768, stream=stream)
        ak.ops.rope_kv_append_q8(qkv, table, 512, pos, slots, q, *cache, 40, 12, 12, 64, blocks, stream=stream)
        ak.ops.attn_decode_paged_q8(q, *cache, tables, klens, out, 40, 1, 12, 12, 64, mb, 0.125, blocks, stream=stream)
        ak.ops.kv_read_q8(*cache, slots, k_out, v_out, 40, 12, 64, blocks, dtype=ak.AK_F32, stream=stream)
    return call, [q8, s8, qkv, q, out, k_out, v_out], x


def test_two_streams_at_once_and_the_same_bits_again(ak, torch_cuda):
    torch = torch_cuda
    works = [_work(ak, torch, s) for s in (1, 2)]
    want = []
    for call, outs, _ in works:
        call(None)
        torch.cuda.synchronize()
        want.append([o.clone() for o in outs])
    streams = [torch.cuda.Stream() for _ in works]
    for _ in range(20):
        for (call, outs, _), s in zip(works, streams):
            call(s.cuda_stream)
    torch.cuda.synchronize()
    for (_, outs, _), w in zip(works, want):
        assert all(torch.equal(a, b) for a, b in zip(outs, w))


def test_captured_and_replayed_on_new_inputs(ak, torch_cuda):
    """Two graphs of the chain, replayed on two streams, on inputs that they have not been captured with."""
    torch = torch_cuda
    works = [_work(ak, torch, s) for s in (3, 4)]
    graphs = []
    for call, outs, _ in works:
        call(None)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            call(torch.cuda.current_stream().cuda_stream)
        graphs.append(graph)
    fresh = [torch.randn(x.shape, device="cuda", generator=_gen(torch, 8 + i)) for i, (_, _, x) in enumerate(works)]
    want = []
    for (call, outs, x), f in zip(works, fresh):
        x.copy_(f)
        call(None)
        torch.cuda.synchronize()
        want.append([o.clone() for o in outs])
        for o in outs:
            o.zero_()
    torch.cuda.synchronize()
    for graph, s in zip(graphs, (torch.cuda.Stream(), torch.cuda.Stream())):
        with torch.cuda.stream(s):
            graph.replay()
    torch.cuda.synchronize()
    for (_, outs, _), w in zip(works, want):
        assert all(torch.equal(a, b) for a, b in zip(outs, w))


# ------------------------------------------------------------------ a decoder layer
def _quantised(y):
    top = y.abs().amax(1, keepdim=True)
    return np.rint(127 * (y / top).cpu().numpy()), top / 127


def test_a_layer_in_8_bits(ak, torch_cuda):
    """A prompt, then a step of two tokens, through a decoder layer of the 8-bit operators as a program would call them, against the same layer in
    64 bits. Both quantise, so an error e before a quantisation moves a value by a whole step (max / 127) with probability |e| / step: a mean square
    of step * |e|, relative to the row's sqrt(c r / 127) for errors of r of a value and c = max * mean|v| / mean v^2, 2.6 for normal values and about 5
    behind the SiLU. The attention's result, off by 2^-8 (bf16): sqrt(2.6 * 2^-8 / 127) = 0.009, which reaches x and through its norm (at most as
    much of x: sqrt(2.6 * 0.009 / 127) = 0.014) the SiLU, whose own rounding adds to it: sqrt(5 * (0.014 + 0.004) / 127) = 0.027. In all
    0.009 + 0.014 + 0.027 = 0.05 of the layer's update in the 2-norm."""
    torch, ops = torch_cuda, ak.ops
    D, H, hd, F, P, n_new = 768, 12, 64, 1280, 37, 2
    g = _gen(torch, 0)
    blocks, ctx = 5, 64
    kp, vp = (torch.zeros(blocks, H, 16, hd, dtype=torch.int8, device="cuda") for _ in range(2))
    ks, vs = (torch.zeros(blocks, H, 16, device="cuda") for _ in range(2))
    tables = torch.tensor([[4, 1, 3, 0]], dtype=torch.int32, device="cuda")
    table = _rope_table(torch, ctx, hd)
    gain1, gain2 = (1 + 0.1 * torch.randn(D, device="cuda", generator=g) for _ in range(2))
    weights = {}
    for name, n, k in (("qkv", 3 * D, D), ("o", D, D), ("up", F, D), ("down", D, F)):
        w = 0.05 * torch.randn(n, k, device="cuda", generator=g)
        q, s = torch.empty(n, k, dtype=torch.int8, device="cuda"), torch.empty(n, device="cuda")
        ops.rmsnorm_q8(w, None, None, q, s, n, k)        # the weights' rows, once
        weights[name] = (q, s)
    slot_of = lambda p: (tables[0, p // 16].long() * 16 + p % 16).int()  # noqa: E731

    def linear(x8, s8, name, out, epi=0):
        wq, ws = weights[name]
        ops.gemm_q8(x8, s8, wq, ws, out, x8.shape[0], wq.shape[0], wq.shape[1], epi)

    def rows8(x, gain=None, bf16=False):
        q, s = torch.empty(x.shape, dtype=torch.int8, device="cuda"), torch.empty(x.shape[0], device="cuda")
        ops.rmsnorm_q8(x, None, gain, q, s, *x.shape, 1e-5, in_dtype=ak.AK_BF16 if bf16 else ak.AK_F32)
        return q, s

    def layer(x, first):
        T = x.shape[0]
        pos = torch.arange(first, first + T, device="cuda", dtype=torch.int32)
        slots = slot_of(pos.long())
        qkv = torch.empty(T, 3 * D, device="cuda")
        linear(*rows8(x, gain1), "qkv", qkv)
        if first == 0:      # the prompt: its cached rows read back, causal attention over them
            q, k, v, a = (torch.empty(T, D, device="cuda") for _ in range(4))
            ops.rope_kv_append_q8(qkv, table, ctx, pos, slots, q, kp, vp, ks, vs, T, H, H, hd, blocks, dtype=ak.AK_F32)
            ops.kv_read_q8(kp, vp, ks, vs, slots, k, v, T, H, hd, blocks, dtype=ak.AK_F32)
            ops.flash_attention(q, k, v, a, T, D, hd, hd ** -0.5)
        else:               # a step of several tokens
            q, a = torch.empty(T, D, device="cuda", dtype=torch.bfloat16), torch.empty(T, D, device="cuda", dtype=torch.bfloat16)
            ops.rope_kv_append_q8(qkv, table, ctx, pos, slots, q, kp, vp, ks, vs, T, H, H, hd, blocks)
            lens = torch.tensor([first + T], dtype=torch.int32, device="cuda")
            ops.attn_decode_paged_q8(q, kp, vp, ks, vs, tables, lens, a, 1, T, H, H, hd, 4, hd ** -0.5, blocks)
        linear(*rows8(a, bf16=first > 0), "o", x, ak.EPI_ADD_F32)
        up = torch.empty(T, F, device="cuda", dtype=torch.bfloat16)
        linear(*rows8(x, gain2), "up", up, ak.EPI_SILU_BF16)
        linear(*rows8(up, bf16=True), "down", x, ak.EPI_ADD_F32)
        return x

    state = {"k": [], "v": []}

    def q64(y):
        q, s = _quantised(y)
        return torch.from_numpy(q).cuda() * s

    def layer64(x, first):
        T = x.shape[0]
        mat = lambda y, name: y @ (weights[name][0].double() * weights[name][1].double()[:, None]).t()  # noqa: E731
        norm = lambda y, gain: y / ((y * y).mean(1, keepdim=True) + 1e-5).sqrt() * gain.double()  # noqa: E731
        qkv = mat(q64(norm(x, gain1)), "qkv").view(T, 3, H, hd)
        cs = table[first:first + T].double()
        q, k = _turn(qkv[:, 0], cs)[0], _turn(qkv[:, 1], cs)[0]
        state["k"].append(q64(k.reshape(T * H, hd)).view(T, H, hd))
        state["v"].append(q64(qkv[:, 2].reshape(T * H, hd)).view(T, H, hd))
        k, v = torch.cat(state["k"]), torch.cat(state["v"])
        s = torch.einsum("thd,jhd->htj", q, k) * hd ** -0.5
        s = s.masked_fill(torch.arange(k.shape[0], device="cuda")[None, None] > (first + torch.arange(T, device="cuda"))[None, :, None], -math.inf)
        a = torch.einsum("htj,jhd->thd", torch.softmax(s, -1), v).reshape(T, D)
        x = x + mat(q64(a), "o")
        u = mat(q64(norm(x, gain2)), "up")
        return x + mat(q64(u * torch.sigmoid(u)), "down")

    for first, T in ((0, P), (P, n_new)):
        x = torch.randn(T, D, device="cuda", generator=g)
        want = layer64(x.double(), first)
        before = x.double()
        got = layer(x.clone(), first).double()
        torch.cuda.synchronize()
        assert float((got - want).norm() / (want - before).norm()) < 0.05
