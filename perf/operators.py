"""Performance cases of the 8-bit operators: a decoder layer whose activations, weights and cache are int8 with f32 scales.

Five operators, each handing its result to the next: the RMS norm (or the plain rows) quantised per token, the product of
8-bit integers with scales per token and output channel, the cache append that rotates and quantises as it writes, reading
cached rows back, and the attention of the newest tokens over that cache. The plain forms say in elementary torch operations
what each computes; `exact` says it again in 64 bits.

Lengths belong to the case, values come from the seed. Buffers, weights and tables are what a serving program keeps.
"""
import math
import random

import torch

own = False

ESZ = {"f32": 4, "bf16": 2}
TORCH = {"f32": torch.float32, "bf16": torch.bfloat16}
DT = {"f32": 0, "bf16": 1}                                                  # ak_dtype
EPI = {"store_f32": 0, "add_f32": 1, "store_bf16": 2, "silu_bf16": 3}       # ak_gemm_epilogue
BS = 16                                                                     # positions per cache block
EPS = 1e-5


def listed():
    return [
        # One decode step of 64 sequences of the 162M model: the residual stream plus an output, normed for the next projection.
        {"name": "norm_decode", "kind": "norm", "rows": 64, "size": 768, "in": "f32", "residual": True, "weight": True},
        # The same over a large prompt of the 1.4B model.
        {"name": "norm_prompt", "kind": "norm", "rows": 16384, "size": 2048, "in": "f32", "residual": True, "weight": True},
        # The SiLU's output of an odd number of prompt tokens, quantised for the ffn-down projection.
        {"name": "rows_prompt", "kind": "norm", "rows": 4001, "size": 8192, "in": "bf16", "residual": False, "weight": False},
        # The fused qkv projection of one decode step of the 162M model.
        {"name": "gemm_decode", "kind": "gemm", "m": 64, "n": 2304, "k": 768, "epilogue": "store_f32", "pad": 0},
        # The ffn-down projection of a prompt, added to the residual stream.
        {"name": "gemm_down", "kind": "gemm", "m": 4001, "n": 2048, "k": 8192, "epilogue": "add_f32", "pad": 0},
        # The ffn-up projection of a large prompt, with its SiLU.
        {"name": "gemm_up", "kind": "gemm", "m": 16384, "n": 8192, "k": 2048, "epilogue": "silu_bf16", "pad": 0},
        # The cache rows of a large prompt, four query heads to a cached head, written and read back.
        {"name": "append_prompt", "kind": "append", "tokens": 16001, "heads": 32, "kv_heads": 8, "head_dim": 128, "dtype": "bf16"},
        # One decode step's tokens written, f32 activations.
        {"name": "append_decode", "kind": "append", "tokens": 64, "heads": 12, "kv_heads": 12, "head_dim": 64, "dtype": "f32"},
        # A long conversation's cached rows read back for a step that works on plain rows.
        {"name": "read_long", "kind": "read", "tokens": 65000, "kv_heads": 8, "head_dim": 128, "dtype": "bf16"},
        # One user of the small model in f32: the shortest call.
        {"name": "attn_one", "kind": "attn", "rows": 1, "q_len": 1, "heads": 5, "kv_heads": 5, "head_dim": 64, "lo": 301, "hi": 301, "dtype": "f32", "lens": 1},
        # A serving batch of the 1.4B model, ragged up to its context.
        {"name": "attn_batch", "kind": "attn", "rows": 64, "q_len": 1, "heads": 16, "kv_heads": 16, "head_dim": 128, "lo": 64, "hi": 4096, "dtype": "bf16", "lens": 2},
        # Two long conversations, four drafted tokens each, four query heads to a cached head.
        {"name": "attn_long", "kind": "attn", "rows": 2, "q_len": 4, "heads": 32, "kv_heads": 8, "head_dim": 128, "lo": 50001, "hi": 65536, "dtype": "bf16", "lens": 3},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["norm", "gemm", "gemm", "append", "read", "attn", "attn"])
    if kind == "norm":
        form = rng.choice(["residual", "plain", "rows"])
        size = _log(rng, 65, 8192)
        rows = _log(rng, 1, min(16384, 33554432 // size))
        return {"kind": kind, "rows": rows, "size": size, "in": rng.choice(["f32", "bf16"]) if form != "residual" else "f32", "residual": form == "residual",
                "weight": form != "rows"}
    if kind == "gemm":
        m, n, k = _log(rng, 1, 8192), _log(rng, 33, 8192), 16 * _log(rng, 4, 512)
        epilogue = rng.choice(list(EPI))
        return {"kind": kind, "m": m, "n": n, "k": k, "epilogue": epilogue, "pad": -n % 8 if rng.random() < 0.7 else 0}
    kv_heads, group, head_dim = rng.choice([1, 2, 4, 5, 8, 12, 16]), rng.choice([1, 1, 2, 4, 8]), rng.choice([32, 64, 64, 96, 128, 128])
    if kind == "append":
        tokens = _log(rng, 1, min(16001, 98000000 // ((group + 2) * kv_heads * head_dim)))
        return {"kind": kind, "tokens": tokens, "heads": group * kv_heads, "kv_heads": kv_heads, "head_dim": head_dim, "dtype": rng.choice(["f32", "bf16"])}
    if kind == "read":
        tokens = _log(rng, 1, min(65000, 66000000 // (kv_heads * head_dim)))
        return {"kind": kind, "tokens": tokens, "kv_heads": kv_heads, "head_dim": head_dim, "dtype": rng.choice(["f32", "bf16"])}
    rows, q_len = _log(rng, 1, 256), rng.choice([1, 1, 1, 2, 4, 5])
    hi = _log(rng, 1, min(65536, 268000000 // (rows * kv_heads * head_dim * q_len)))
    return {"kind": kind, "rows": rows, "q_len": q_len, "heads": group * kv_heads, "kv_heads": kv_heads, "head_dim": head_dim, "lo": rng.randint(1, hi), "hi": hi,
            "dtype": rng.choice(["f32", "bf16"]), "lens": rng.randint(1, 1 << 20)}


# ------------------------------------------------------------------ inputs
def _lens(case):
    r = random.Random(case["lens"])
    return [r.randint(case["lo"], case["hi"]) for _ in range(case["rows"])]


def _rows_to_int8(y):
    """Rows of f32 as int8 and scales, for inputs that a program has in hand already quantised."""
    s = y.abs().amax(-1, keepdim=True) / 127
    return torch.round(y / s).to(torch.int8), s.squeeze(-1)


def _pools(g, blocks, kv_heads, head_dim):
    """Two pools of cached rows and their scales, a few blocks at a time."""
    dev = g.device
    pools = [torch.empty((blocks, kv_heads, BS, head_dim), dtype=torch.int8, device=dev) for _ in range(2)]
    scales = [torch.empty((blocks, kv_heads, BS), dtype=torch.float32, device=dev) for _ in range(2)]
    step = max(1, (1 << 26) // (kv_heads * BS * head_dim))
    for b in range(0, blocks, step):
        for p, s in zip(pools, scales):
            y = torch.randn((min(step, blocks - b), kv_heads, BS, head_dim), generator=g, device=dev)
            p[b:b + step], s[b:b + step] = _rows_to_int8(y)
    return pools, scales


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev)
    g.manual_seed(seed)

    def randn(*shape):
        return torch.randn(shape, generator=g, device=dev)

    s = {"case": case}
    if case["kind"] == "norm":
        rows, size = case["rows"], case["size"]
        s["x"] = randn(rows, size).to(TORCH[case["in"]])
        s["residual"] = randn(rows, size) if case["residual"] else None
        s["weight"] = 1 + 0.1 * randn(size) if case["weight"] else None
        s["q"] = torch.empty((rows, size), dtype=torch.int8, device=dev)
        s["scales"] = torch.empty(rows, device=dev)
        s["values"] = torch.empty((rows, size), dtype=torch.bfloat16, device=dev)
    elif case["kind"] == "gemm":
        m, n, k = case["m"], case["n"], case["k"]
        s["a"], s["a_scales"] = _rows_to_int8(randn(m, k))
        s["wt"], s["w_scales"] = _rows_to_int8(0.02 * randn(n, k))
        f32 = case["epilogue"].endswith("f32")
        ld = n + case["pad"]
        s["c"] = randn(m, ld) if case["epilogue"] == "add_f32" else torch.zeros((m, ld), dtype=torch.float32 if f32 else torch.bfloat16, device=dev)
    elif case["kind"] in ("append", "read"):
        tokens, kv_heads, hd = case["tokens"], case["kv_heads"], case["head_dim"]
        blocks = -(-tokens // BS) + 3
        s["slots"] = torch.randperm(blocks * BS, generator=g, device=dev)[:tokens].to(torch.int32)
        s["blocks"] = blocks
        out = TORCH[case["dtype"]] if case["kind"] == "read" else torch.bfloat16
        s["k_out"] = torch.empty((tokens, kv_heads * hd), dtype=out, device=dev)
        s["v_out"] = torch.empty((tokens, kv_heads * hd), dtype=out, device=dev)
        if case["kind"] == "read":
            (s["k_pool"], s["v_pool"]), (s["k_scales"], s["v_scales"]) = _pools(g, blocks, kv_heads, hd)
            return s
        s["qkv"] = randn(tokens, (case["heads"] + 2 * kv_heads) * hd)
        s["rope_len"] = 32768
        inv = 10000.0 ** (-torch.arange(0, hd, 2, device=dev, dtype=torch.float64) / hd)
        angle = torch.arange(s["rope_len"], device=dev, dtype=torch.float64)[:, None] * inv
        s["rope"] = torch.stack([angle.cos(), angle.sin()], -1).float().contiguous()
        s["positions"] = torch.randint(0, s["rope_len"], (tokens,), generator=g, device=dev, dtype=torch.int32)
        s["q_out"] = torch.empty((tokens, case["heads"] * hd), dtype=TORCH[case["dtype"]], device=dev)
        for name in ("k", "v"):
            s[name + "_pool"] = torch.zeros((blocks, kv_heads, BS, hd), dtype=torch.int8, device=dev)
            s[name + "_scales"] = torch.zeros((blocks, kv_heads, BS), device=dev)
    else:
        rows, kv_heads, hd = case["rows"], case["kv_heads"], case["head_dim"]
        lens = _lens(case)
        per = [-(-n // BS) for n in lens]
        s["blocks"], s["max_blocks"] = sum(per) + 2, max(per)
        order = torch.randperm(s["blocks"], generator=g, device=dev).to(torch.int32)
        have = torch.arange(s["max_blocks"], device=dev)[None, :] < torch.tensor(per, device=dev)[:, None]
        s["tables"] = torch.full((rows, s["max_blocks"]), -1, dtype=torch.int32, device=dev)
        s["tables"][have] = order[:sum(per)]
        s["lens"] = torch.tensor(lens, dtype=torch.int32, device=dev)
        (s["k_pool"], s["v_pool"]), (s["k_scales"], s["v_scales"]) = _pools(g, s["blocks"], kv_heads, hd)
        s["q"] = (2 * randn(rows * case["q_len"], case["heads"] * hd)).to(TORCH[case["dtype"]])
        s["out"] = torch.empty_like(s["q"])
    return s


# ------------------------------------------------------------------ the framework's calls
def _ops():
    import __graft_entry__ as entry
    return entry.load_package().ops


def _run_own(s):
    ops, c = _ops(), s["case"]
    if c["kind"] == "norm":
        ops.rmsnorm_q8(s["x"], s["residual"], s["weight"], s["q"], s["scales"], c["rows"], c["size"], EPS, in_dtype=DT[c["in"]])
        torch.mul(s["q"], s["scales"][:, None], out=s["values"])   # what the 8 bits stand for
        return {"values": s["values"], "scales": s["scales"], **({"x": s["x"]} if c["residual"] else {})}
    if c["kind"] == "gemm":
        ops.gemm_q8(s["a"], s["a_scales"], s["wt"], s["w_scales"], s["c"], c["m"], c["n"], c["k"], EPI[c["epilogue"]], ldc=c["n"] + c["pad"])
        return s["c"][:, :c["n"]]
    if c["kind"] == "attn":
        ops.attn_decode_paged_q8(s["q"], s["k_pool"], s["v_pool"], s["k_scales"], s["v_scales"], s["tables"], s["lens"], s["out"], c["rows"], c["q_len"],
                                 c["heads"], c["kv_heads"], c["head_dim"], s["max_blocks"], c["head_dim"] ** -0.5, s["blocks"], dtype=DT[c["dtype"]])
        return s["out"]
    out = {}
    if c["kind"] == "append":
        ops.rope_kv_append_q8(s["qkv"], s["rope"], s["rope_len"], s["positions"], s["slots"], s["q_out"], s["k_pool"], s["v_pool"], s["k_scales"],
                              s["v_scales"], c["tokens"], c["heads"], c["kv_heads"], c["head_dim"], s["blocks"], dtype=DT[c["dtype"]])
        out = {"q": s["q_out"], "k_scales": s["k_scales"], "v_scales": s["v_scales"]}
    ops.kv_read_q8(s["k_pool"], s["v_pool"], s["k_scales"], s["v_scales"], s["slots"], s["k_out"], s["v_out"], c["tokens"], c["kv_heads"], c["head_dim"],
                   s["blocks"], dtype=DT[c["dtype"]] if c["kind"] == "read" else DT["bf16"])
    return {**out, "k": s["k_out"], "v": s["v_out"]}


# ------------------------------------------------------------------ the plain forms
def _quantised(y):
    """(values -127..127, scales) of the rows of y, in f32."""
    top = y.abs().amax(-1, keepdim=True)
    return torch.round(y * (127 / top.clamp(min=1e-36))), (top / 127).squeeze(-1)


def _rotated(x, cs):
    """Adjacent pairs of every head turned by their position's angle. x [tokens, heads, head_dim], cs [tokens, 1, head_dim / 2, 2]."""
    a, b = x[..., 0::2], x[..., 1::2]
    return torch.stack([a * cs[..., 0] - b * cs[..., 1], a * cs[..., 1] + b * cs[..., 0]], -1).flatten(-2)


def run(s):
    if own:
        return _run_own(s)
    c = s["case"]
    if c["kind"] == "norm":
        h = s["x"]
        if c["residual"]:
            h.add_(s["residual"])
        y = h.float()
        if c["weight"]:
            y = y * torch.rsqrt(y.square().mean(-1, keepdim=True) + EPS) * s["weight"]
        q, scales = _quantised(y)
        return {"values": (q * scales[:, None]).bfloat16(), "scales": scales, **({"x": h} if c["residual"] else {})}
    if c["kind"] == "gemm":
        y = torch.matmul(s["a"].float(), s["wt"].float().t()) * s["a_scales"][:, None] * s["w_scales"]
        if c["epilogue"] == "silu_bf16":
            y = y / (1 + torch.exp(-y))
        out = s["c"][:, :c["n"]]
        return out.add_(y) if c["epilogue"] == "add_f32" else out.copy_(y)
    if c["kind"] == "attn":
        rows, q_len, kv_heads, hd = c["rows"], c["q_len"], c["kv_heads"], c["head_dim"]
        length = s["max_blocks"] * BS
        table = s["tables"].clamp(min=0).long()

        def cached(pool, scales):   # [rows, kv_heads, length, head_dim] in f32
            y = pool[table].float() * scales[table][..., None]
            return y.transpose(1, 2).reshape(rows, kv_heads, length, hd)

        q = s["q"].float().view(rows, q_len, kv_heads, -1, hd).permute(0, 2, 3, 1, 4).reshape(rows, kv_heads, -1, hd)
        score = torch.matmul(q, cached(s["k_pool"], s["k_scales"]).transpose(2, 3)) * hd ** -0.5
        at = s["lens"].long()[:, None] - q_len + torch.arange(q_len, device=q.device)                  # position of each query
        seen = torch.arange(length, device=q.device)[None, None, :] <= at[:, :, None]                   # [rows, q_len, length]
        seen = seen[:, None, None].expand(rows, kv_heads, q.shape[2] // q_len, q_len, length).reshape(score.shape)
        score = score.masked_fill(~seen, -math.inf)
        top = score.amax(-1, keepdim=True).clamp(min=-3e38)
        p = torch.exp(score - top)
        p = p / p.sum(-1, keepdim=True).clamp(min=1e-30)
        o = torch.matmul(p, cached(s["v_pool"], s["v_scales"]))
        o = o.view(rows, kv_heads, -1, q_len, hd).permute(0, 3, 1, 2, 4).reshape(rows * q_len, -1)
        return s["out"].copy_(o)
    tokens, kv_heads, hd = c["tokens"], c["kv_heads"], c["head_dim"]
    slots = s["slots"].long()
    block, place = slots // BS, slots % BS
    out = {}
    if c["kind"] == "append":
        x = s["qkv"].view(tokens, -1, hd)
        cs = s["rope"][s["positions"].long()][:, None]
        turned = _rotated(x[:, :-kv_heads], cs)
        for name, y in (("k", turned[:, c["heads"]:]), ("v", x[:, -kv_heads:])):
            q, scales = _quantised(y)
            s[name + "_pool"][block, :, place] = q.to(torch.int8)
            s[name + "_scales"][block, :, place] = scales
        out = {"q": s["q_out"].copy_(turned[:, :c["heads"]].reshape(tokens, -1)), "k_scales": s["k_scales"], "v_scales": s["v_scales"]}
    for name in ("k", "v"):
        y = s[name + "_pool"][block, :, place].float() * s[name + "_scales"][block, :, place][..., None]
        out[name] = s[name + "_out"].copy_(y.reshape(tokens, -1))
    return out


# ------------------------------------------------------------------ 64 bits
def exact(case, seed):
    c, s = case, prepare(case, seed)
    if c["kind"] == "norm":
        h = s["x"].double()
        if c["residual"]:
            h += s["residual"].double()
        scales = torch.empty(c["rows"], dtype=torch.float64, device=h.device)
        values = torch.empty_like(h)
        for r in range(0, c["rows"], 1024):
            y = h[r:r + 1024]
            if c["weight"]:
                y = y / ((y ** 2).sum(1) / c["size"] + EPS).sqrt()[:, None] * s["weight"].double()
            scales[r:r + 1024] = y.abs().max(1).values / 127
            values[r:r + 1024] = (y / scales[r:r + 1024, None]).round() * scales[r:r + 1024, None]
        return {"values": values, "scales": scales, **({"x": h} if c["residual"] else {})}
    if c["kind"] == "gemm":
        out = torch.empty((c["m"], c["n"]), dtype=torch.float64, device=s["a"].device)
        w = s["wt"].double() * s["w_scales"].double()[:, None]
        for r in range(0, c["m"], 2048):
            y = (s["a"][r:r + 2048].double() * s["a_scales"][r:r + 2048, None].double()) @ w.T
            if c["epilogue"] == "silu_bf16":
                y = y * torch.sigmoid(y)
            if c["epilogue"] == "add_f32":
                y += s["c"][r:r + 2048, :c["n"]].double()
            out[r:r + 2048] = y
        return out
    if c["kind"] == "attn":
        q_len, hd, group = c["q_len"], c["head_dim"], c["heads"] // c["kv_heads"]
        out = torch.zeros((c["rows"], q_len, c["heads"], hd), dtype=torch.float64, device=s["q"].device)
        q = s["q"].double().view(c["rows"], q_len, c["heads"], hd)
        for r, n in enumerate(_lens(c)):
            ids = s["tables"][r, :-(-n // BS)].long()
            k, v = ((s[p + "_pool"][ids].double() * s[p + "_scales"][ids].double().unsqueeze(-1)).permute(1, 0, 2, 3).flatten(1, 2)[:, :n] for p in "kv")
            for i in range(q_len):
                m = n - q_len + i + 1
                if m > 0:
                    w = torch.softmax(torch.einsum("hgd,hjd->hgj", q[r, i].view(-1, group, hd), k[:, :m]) / math.sqrt(hd), -1)
                    out[r, i] = torch.einsum("hgj,hjd->hgd", w, v[:, :m]).reshape(-1, hd)
        return out.view(c["rows"] * q_len, -1)
    block, place = s["slots"].long() // BS, s["slots"].long() % BS
    if c["kind"] == "read":
        return {n: (s[n + "_pool"].double() * s[n + "_scales"].double().unsqueeze(-1))[block, :, place].flatten(1) for n in "kv"}
    x = s["qkv"].double().view(c["tokens"], -1, c["head_dim"])
    angle = torch.view_as_complex(s["rope"].double())[s["positions"].long()][:, None]
    turned = torch.view_as_real(torch.view_as_complex(x.unflatten(-1, (-1, 2)).contiguous()) * angle).flatten(-2)
    out = {"q": turned[:, :c["heads"]].flatten(1)}
    for name, y in (("k", turned[:, c["heads"]:c["heads"] + c["kv_heads"]]), ("v", x[:, c["heads"] + c["kv_heads"]:])):
        step = y.abs().amax(-1) / 127
        out[name] = ((y / step[..., None]).round() * step[..., None]).flatten(1)
        out[name + "_scales"] = s[name + "_scales"].double()
        out[name + "_scales"][block, :, place] = step
    return out


# ------------------------------------------------------------------ what a pass cannot do without
def work(case):
    c = case
    if c["kind"] == "norm":
        e = c["rows"] * c["size"]
        return {"bytes": e * (ESZ[c["in"]] + 1 + (8 if c["residual"] else 0)) + 4 * c["rows"] + (4 * c["size"] if c["weight"] else 0), "flops": 8 * e}
    if c["kind"] == "gemm":
        m, n, k = c["m"], c["n"], c["k"]
        out = {"store_f32": 4, "add_f32": 8, "store_bf16": 2, "silu_bf16": 2}[c["epilogue"]]
        return {"bytes": m * k + n * k + 4 * (m + n) + out * m * n, "flops": 2 * m * n * k}
    cached = c["kv_heads"] * (2 * c["head_dim"] + 8)
    if c["kind"] == "attn":
        total = sum(_lens(c))
        q = c["rows"] * c["q_len"] * c["heads"] * c["head_dim"]
        return {"bytes": total * cached + 2 * q * ESZ[c["dtype"]] + 4 * total // BS, "flops": 4 * total * c["q_len"] * c["heads"] * c["head_dim"]}
    row = c["tokens"] * c["kv_heads"] * c["head_dim"]
    if c["kind"] == "read":
        return {"bytes": c["tokens"] * (cached + 4) + 2 * row * ESZ[c["dtype"]], "flops": 2 * row}
    # written, and read back as bf16
    q = c["tokens"] * c["heads"] * c["head_dim"]
    return {"bytes": q * (4 + ESZ[c["dtype"]]) + 2 * row * 4 + c["tokens"] * (2 * cached + 8) + 2 * row * 2, "flops": 6 * q + 12 * row}
