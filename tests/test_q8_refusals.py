"""CPU and GPU: what the 8-bit operators refuse. Every check of an argument comes before the first CUDA call, so these run without a GPU; the
pointers are never followed."""
import ctypes as C

import pytest

P = 0x10000          # a pointer aligned to everything
F32, BF16 = 0, 1


def _call(ak, name, good, **bad):
    kw = dict(good)
    kw.update(bad)
    with pytest.raises(ak.AkashaError) as e:
        getattr(ak.ops, name)(**kw)
    return e.value


NORM = dict(x=P, residual=None, weight=P, q=P, scales=P, rows=3, size=64)
GEMM = dict(a=P, a_scales=P, wt=P, w_scales=P, c=P, m=3, n=5, k=32)
APPEND = dict(qkv=P, rope_table=P, rope_len=8, positions=P, slots=P, q_out=P, k_pool=P, v_pool=P, k_scales=P, v_scales=P, tokens=3, heads=4, kv_heads=2,
              head_dim=64, pool_blocks=4)
READ = dict(k_pool=P, v_pool=P, k_scales=P, v_scales=P, slots=P, k_out=P, v_out=P, tokens=3, kv_heads=2, head_dim=64, pool_blocks=4)
ATTN = dict(q=P, k_pool=P, v_pool=P, k_scales=P, v_scales=P, block_tables=P, kv_lens=P, out=P, rows=2, q_len=1, heads=4, kv_heads=2, head_dim=64,
            max_blocks_per_seq=4, scale=0.125, pool_blocks=4)
CACHE = [("k_pool", P + 8), ("v_scales", P + 4), ("kv_heads", 0), ("kv_heads", 3), ("heads", 0), ("head_dim", 48), ("head_dim", 256), ("head_dim", 0),
         ("pool_blocks", 0), ("pool_blocks", (1 << 27) + 1), ("dtype", 2), ("k_pool", 0), ("v_scales", 0)]


@pytest.mark.parametrize("name,good,bad", [("rmsnorm_q8", NORM, b) for b in [
    dict(x=0), dict(q=0), dict(scales=0), dict(in_dtype=2), dict(residual=P, in_dtype=BF16), dict(x=P + 2), dict(weight=P + 1), dict(scales=P + 2),
    dict(residual=P + 2), dict(size=(1 << 31) - 1), dict(rows=1 << 31)]] + [("gemm_q8", GEMM, b) for b in [
        dict(a=0), dict(a_scales=0), dict(wt=0), dict(w_scales=0), dict(c=0), dict(k=0), dict(k=8), dict(k=40), dict(k=131072), dict(epilogue=4), dict(ldc=4),
        dict(a=P + 8), dict(wt=P + 1), dict(c=P + 4), dict(a_scales=P + 2), dict(m=65535 * 128 + 1), dict(n=(1 << 30) + 1)]] + [
            ("rope_kv_append_q8", APPEND, {k: v}) for k, v in CACHE + [
                ("qkv", 0), ("rope_table", 0), ("positions", 0), ("slots", 0), ("q_out", 0), ("rope_len", 0), ("rope_len", 1 << 31), ("qkv", P + 4), ("rope_table", P + 8), ("q_out", P + 2),
                ("slots", P + 2)]] + [
                    ("kv_read_q8", READ, b) for b in [{k: v} for k, v in CACHE if k != "heads" and (k, v) != ("kv_heads", 3)] + [
                        dict(k_out=None, v_out=None), dict(slots=0), dict(k_out=P + 8), dict(v_out=P + 4), dict(slots=P + 1)]] + [
                            ("attn_decode_paged_q8", ATTN, {k: v}) for k, v in CACHE + [
                                ("q", 0), ("out", 0), ("block_tables", 0), ("kv_lens", 0), ("q_len", 0), ("q_len", (1 << 22) + 1), ("q_len", (1 << 32) - 1), ("n_splits", 17), ("max_blocks_per_seq", 0),
                                ("max_blocks_per_seq", (1 << 26) + 1), ("q", P + 8), ("out", P + 2), ("kv_lens", P + 2)]])
def test_refused(ak, name, good, bad):
    e = _call(ak, name, good, **bad)
    assert e.kind in ("InvalidArg", "Unsupported") and "ak_" + name in str(e)


@pytest.mark.parametrize("name,good", [("rmsnorm_q8", dict(NORM, rows=0)), ("rmsnorm_q8", dict(NORM, size=0)), ("gemm_q8", dict(GEMM, m=0)), ("gemm_q8", dict(GEMM, n=0)),
                                       ("rope_kv_append_q8", dict(APPEND, tokens=0)), ("kv_read_q8", dict(READ, tokens=0)), ("attn_decode_paged_q8", dict(ATTN, rows=0))])
def test_nothing_to_do(ak, name, good):
    getattr(ak.ops, name)(**good)


def test_block_size_is_16(ak):
    p = ak.AttnQ8Params(2, 1, 4, 2, 64, 32, 4, 0.125, F32, 0, 4)
    assert ak.lib().ak_attn_decode_paged_q8(None, P, P, P, P, P, P, P, P, p) == 103
    assert ak.lib().ak_kv_read_q8(None, P, P, P, P, P, P, P, 3, 2, 64, 8, F32, 4) == 103
    assert ak.lib().ak_rope_kv_append_q8(None, P, P, 8, P, P, P, P, P, P, P, 3, 4, 2, 64, 8, F32, 4) == 103


def test_params_match_the_header(ak):
    import test_abi_and_host as abi
    assert [f for f, _ in ak.AttnQ8Params._fields_] == abi._struct_fields("ak_attn_q8_params")
    assert C.sizeof(ak.AttnQ8Params) == 4 * len(ak.AttnQ8Params._fields_)


def test_tensors_that_are_not_what_the_kernel_reads(ak):
    """A tensor of another type, with strides, too short or on the CPU is refused by name before the library is called."""
    import torch
    for bad in (torch.zeros(3, 64, dtype=torch.float32), torch.zeros(3, 64, dtype=torch.float16)):
        e = _call(ak, "rmsnorm_q8", NORM, x=bad)
        assert e.kind == "InvalidArg" and "x has to be" in str(e)
    if torch.cuda.is_available():
        x = torch.zeros(64, 6, device="cuda")
        for bad in (x.t()[:3], x[:2], x.double()):
            assert "x has to be" in str(_call(ak, "rmsnorm_q8", NORM, x=bad))
    assert "q is missing" in str(_call(ak, "attn_decode_paged_q8", ATTN, q=None))
