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


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("rows,size,offset", FORMS + [(700, 14001, 0), (130, 3, 0)])
def test_rows_take_three_roundings(ak, torch_cuda, dtype, rows, size, offset):
    """q = rint(y (127 (1 / max|y|))) with each of the operations rounded to f32, half-way cases to even: the same integers whatever kernel a size or an
    alignment picks. Values of bf16 are often half-way."""
    torch = torch_cuda
    dt, tdt = _dt(ak, torch, dtype)
    x = torch.randn(rows, size, device="cuda", generator=_gen(torch, rows + size)).to(tdt)
    x = x * torch.ldexp(torch.ones(rows, 1, device="cuda"), torch.arange(rows, device="cuda")[:, None] % 200 - 80).to(tdt)
    x[-1] = x[-1].sign() * 3.0e38        # the largest numbers
    x = _at(torch, x, offset)
    q, scales = torch.full((rows, size), 77, dtype=torch.int8, device="cuda"), torch.full((rows,), 7.0, device="cuda")
    ak.ops.rmsnorm_q8(x, None, None, q, scales, rows, size, in_dtype=dt)
    torch.cuda.synchronize()
    y = x.float()
    top = y.abs().amax(1, keepdim=True)
    inv = (top * 0.25).reciprocal() * 31.75        # (the quarter: 1 / 3e38 is subnormal)
    assert torch.equal(q.float(), torch.round(y * inv))
    assert torch.equal(scales[:, None], top * torch.tensor(1.0 / 127.0, dtype=torch.float32, device="cuda"))


def test_half_way_values_go_to_the_even_integer(ak, torch_cuda):
    """max|y| = 127 times a power of two: the quotients are the values, exactly."""
    torch = torch_cuda
    y = torch.arange(-254, 255, device="cuda").float() / 2
    for dtype in ("f32", "bf16"):
        dt, tdt = _dt(ak, torch, dtype)
        for power in (-90, -3, 0, 60):
            x = torch.ldexp(y, torch.tensor(power, device="cuda")).to(tdt).expand(3, -1).contiguous()
            q, scales = torch.full(x.shape, 77, dtype=torch.int8, device="cuda"), torch.full((3,), 7.0, device="cuda")
            ak.ops.rmsnorm_q8(x, None, None, q, scales, 3, x.shape[1], in_dtype=dt)
            torch.cuda.synchronize()
            assert torch.equal(q.float(), torch.round(y).expand(3, -1))


@pytest.mark.parametrize("heads,kv_heads,hd", [(2, 1, 32), (5, 5, 64), (6, 3, 96), (4, 2, 128)])
def test_append_takes_three_roundings(ak, torch_cuda, heads, kv_heads, hd):
    """The same of the cache's rows: values as they are, keys rotated with one rounding per operation; half of the values are those of bf16."""
    torch = torch_cuda
    tokens, blocks = 333, 30
    g = _gen(torch, hd)
    x = torch.randn(tokens, heads + 2 * kv_heads, hd, device="cuda", generator=g)
    x[::2] = x[::2].bfloat16().float()
    table = ops8._rope_table(torch, 50, hd)
    pos = torch.randint(0, 50, (tokens,), device="cuda", generator=g, dtype=torch.int32)
    slots = torch.randperm(blocks * 16, device="cuda", generator=g)[:tokens].to(torch.int32)
    kp, vp, ks, vs = ops8._cache(torch, blocks, kv_heads, hd, 1)
    q = torch.empty(tokens, heads * hd, device="cuda")
    ak.ops.rope_kv_append_q8(x, table, 50, pos, slots, q, kp, vp, ks, vs, tokens, heads, kv_heads, hd, blocks, dtype=ak.AK_F32)
    torch.cuda.synchronize()
    a, b, c, s = x[..., 0::2], x[..., 1::2], table[pos.long()][:, None, :, 0], table[pos.long()][:, None, :, 1]
    turned = torch.stack([a * c - b * s, a * s + b * c], -1).flatten(-2)
    assert torch.equal(q.view(tokens, heads, hd), turned[:, :heads])
    at = slots.long()
    for pool, scales, y in ((kp, ks, turned[:, heads:heads + kv_heads]), (vp, vs, x[:, heads + kv_heads:])):
        top = y.abs().amax(-1, keepdim=True)
        assert torch.equal(pool[at // 16, :, at % 16].float(), torch.round(y * (top.reciprocal() * 127)))
        assert torch.equal(scales[at // 16, :, at % 16][..., None], top * torch.tensor(1.0 / 127.0, dtype=torch.float32, device="cuda"))


# ------------------------------------------------------------------ product
@pytest.mark.parametrize("epi", [0, 1, 2, 3])
@pytest.mark.parametrize("n,k,pad", [(768, 2304, 0), (2048, 2048, 0), (777, 1024, 0), (300, 4096, 5), (1002, 2048, 0)])
def test_product_rows_do_not_depend_on_the_batch(ak, torch_cuda, epi, n, k, pad):
    """A row alone, in decode batches, in prompts: the same bits with every epilogue and any pitch, whatever kernel and split it ran on."""
    torch = torch_cuda
    g = _gen(torch, n + k)
    most, ld = 3000, n + pad
    a, wt = _int8(torch, (most, k), g), _int8(torch, (n, k), g)
    sa, sw = 0.01 + torch.rand(most, device="cuda", generator=g), (0.01 + torch.rand(n, device="cuda", generator=g)) / k
    start = torch.randn(most, ld, device="cuda", generator=g).to(torch.float32 if epi < 2 else torch.bfloat16)

    def product(m):
        c = start[:m].clone()
        ak.ops.gemm_q8(a[:m], sa[:m], wt, sw, c, m, n, k, epi, ldc=ld)
        return c

    full = product(most)
    for m in (1, 3, 8, 17, 64, 100, 128, 200, 500, 1000, 2048):
        assert torch.equal(product(m), full[:m]), m
    if epi < 2:    # the sum to f32, two products, and the addition, each rounded
        y = (a.double() @ wt.double().t()).float() * sa[:, None] * sw
        assert torch.equal(full[:, :n], start[:, :n] + y if epi == 1 else y)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("rows,size,offset", FORMS + [(600, 200, 1)])
@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("eps", [0.0, 1e-5])
def test_norm_at_the_ends_of_its_range(ak, torch_cuda, dtype, rows, size, offset, residual, eps):
    """Mean squares from 1e-36 on up to sums of f32's largest number are ordinary. Outside (values of 1e20, or 1e-20 without eps) the scale is NaN, not that of
    another row or a zero, and nothing else of the call is. Zeros are zeros, without eps too."""
    torch = torch_cuda
    if residual and dtype == "bf16":
        pytest.skip("a residual is added to f32 rows only")
    dt, tdt = _dt(ak, torch, dtype)
    kind = torch.arange(rows, device="cuda") % 8
    power = torch.tensor([0, 66, -83, 120, 0, -66, 54, -56], device="cuda")[kind]       # 2^66 = 7e19, 2^-83 = 1e-25, 2^-56 = 1.4e-17
    g = _gen(torch, size + rows)
    x = torch.randn(rows, size, device="cuda", generator=g)
    x[kind == 4] = 0
    res = 0.5 * x.flip(1) if residual else None
    x = torch.ldexp(x, power[:, None]).to(tdt)
    w = 1 + 0.2 * torch.randn(size, device="cuda", generator=g)
    if res is not None:
        res = _at(torch, torch.ldexp(res, power[:, None]), offset)
    x, w = _at(torch, x, offset), _at(torch, w, offset)
    h = x + res if res is not None else x.clone()
    q, scales = torch.full((rows, size), 77, dtype=torch.int8, device="cuda"), torch.full((rows,), 7.0, device="cuda")
    ak.ops.rmsnorm_q8(x, res, w, q, scales, rows, size, eps, in_dtype=dt)
    torch.cuda.synchronize()
    assert torch.equal(x, h)
    none, lost = kind == 4, (kind == 1) | (kind == 3)
    if eps == 0:
        lost |= (kind == 2) | (kind == 5)
    assert (q[none] == 0).all() and (scales[none] == 0).all()
    assert (q[lost] == 0).all() and scales[lost].isnan().all()
    kept = ~(none | lost)
    _check_rows(torch, _normed(torch, h, w, eps)[kept], _norm_error(size), q[kept], scales[kept])


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("size", [1, 2, 3, 5, 6, 7, 9, 11])
def test_norm_of_rows_about_as_short_as_a_vector(ak, torch_cuda, dtype, residual, size):
    """Several rows to 16 bytes: a row's vectors would reach over its neighbours, and over the end of the buffer for more rows than the last."""
    torch = torch_cuda
    if residual and dtype == "bf16":
        pytest.skip("a residual is added to f32 rows only")
    dt, tdt = _dt(ak, torch, dtype)
    for rows in (1, 2, 3, 4, 5, 7, 9, 150, 1201):
        g = _gen(torch, 10 * rows + size)
        x = torch.randn(rows, size, device="cuda", generator=g).to(tdt)
        res = torch.randn(rows, size, device="cuda", generator=g) if residual else None
        w = 1 + 0.2 * torch.randn(size, device="cuda", generator=g)
        h = x + res if residual else x.clone()
        q, scales = torch.full((rows, size), 77, dtype=torch.int8, device="cuda"), torch.full((rows,), 7.0, device="cuda")
        ak.ops.rmsnorm_q8(x, res, w, q, scales, rows, size, in_dtype=dt)
        torch.cuda.synchronize()
        assert torch.equal(x, h)
        _check_rows(torch, _normed(torch, h, w, 1e-5), _norm_error(size), q, scales)


# ------------------------------------------------------------------ attention
@pytest.mark.parametrize("dtype,q_len,heads,kv_heads,power", [("bf16", 6, 2, 2, 30), ("bf16", 8, 4, 2, 60), ("bf16", 2, 4, 2, 60), ("f32", 2, 2, 2, 60),
                                                              ("f32", 7, 2, 1, 60)])
@pytest.mark.parametrize("hd", [32, 64, 96, 128])
@pytest.mark.parametrize("n_splits", [1, 2])
def test_attn_value_that_a_later_token_brings(ak, torch_cuda, dtype, q_len, heads, kv_heads, hd, power, n_splits):
    """The newest token's value is 2^power times the others: the queries before it do not see it, and their results are as without it."""
    torch = torch_cuda
    dt, tdt = _dt(ak, torch, dtype)
    lens = [q_len, 13, 16, 31, 200]
    cache, tables, klens, blocks, mb = ops8._attn_case(torch, lens, kv_heads, hd, 5)
    q = torch.randn(len(lens) * q_len, heads * hd, device="cuda", generator=_gen(torch, 2)).to(tdt)
    for r, n in enumerate(lens):
        cache[3][tables[r, (n - 1) // 16].long(), :, (n - 1) % 16] *= 2.0 ** power
    out = torch.full_like(q, 7.0)
    ak.ops.attn_decode_paged_q8(q, *cache, tables, klens, out, len(lens), q_len, heads, kv_heads, hd, mb, hd ** -0.5, blocks, dtype=dt, n_splits=n_splits)
    torch.cuda.synchronize()
    ops8._attn_check(torch, out.view(len(lens), q_len, -1)[:, :q_len - 1].contiguous(), q.view(len(lens), q_len, -1)[:, :q_len - 1].contiguous(), cache, tables,
                     [n - 1 for n in lens], q_len - 1, heads, kv_heads, hd, hd ** -0.5, dtype, blocks)
