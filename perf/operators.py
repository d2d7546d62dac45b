"""Cases of the 8-bit floating-point linears and the windowed attention, for measurement.

Three operators, as the entry points of include/da3b.h offer them:

* linear: rows of 16-bit activations are quantised to e4m3 with one power-of-two scale for
  each row and 128 columns (da3b_quantize_fp8), then multiplied by weights held the same way
  (da3b_linear_fp8, or da3b_linear_fp8_resid_f32 onto an f32 residual stream);
* mlp: the second half of a ViT block on an f32 residual row: LayerNorm straight into e4m3
  (da3b_layernorm_fp8), the first linear with GELU whose output is quantised by the product's
  own epilogue (da3b_linear_fp8_q), and the second linear;
* attn: softmax attention of the last queries of a sequence over its keys, where a query sees
  a window of keys around its own position and the first few keys (da3b_attention_window).

`own` chooses between the plain torch forms and the library's entry points.
"""
import ctypes
import math

import torch

own = False

_DT = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
_CODE = {"f16": 0, "bf16": 1, "f32": 2}
EPS = 1e-6


# ---------------------------------------------------------------------------- cases
def listed():
    return [
        # one token's projection, the smallest call: launch latency and 4 MB of weights
        {"name": "linear_one_row", "op": "linear", "M": 1, "K": 1024, "N": 4096, "x": "f16", "act": "none", "out": "f16"},
        # nothing is a multiple of a tile: a ragged last block of the reduction, odd columns
        {"name": "linear_odd", "op": "linear", "M": 333, "K": 1000, "N": 771, "x": "bf16", "act": "relu", "out": "bf16"},
        # fc1 of ViT-L for one image of 518 x 518 (1370 tokens)
        {"name": "linear_fc1_1img", "op": "linear", "M": 1370, "K": 1024, "N": 4096, "x": "f16", "act": "gelu", "out": "f16"},
        # fc2 of ViT-L for 8 images, onto the residual stream
        {"name": "linear_fc2_8img", "op": "linear", "M": 10960, "K": 4096, "N": 1024, "x": "f16", "act": "none", "out": "resid"},
        # fc1 of ViT-L for 64 images, the largest product
        {"name": "linear_fc1_64img", "op": "linear", "M": 87680, "K": 1024, "N": 4096, "x": "f16", "act": "none", "out": "f16"},
        # the MLP half of a ViT-L block, one image and 16 images
        {"name": "mlp_1img", "op": "mlp", "M": 1370, "D": 1024, "H": 4096},
        {"name": "mlp_16img", "op": "mlp", "M": 21920, "D": 1024, "H": 4096},
        # one new token (a camera token) over 8 cached views of 504 x 504 (1297 tokens each):
        # it sees the first view and the last four
        {"name": "attn_one_token", "op": "attn", "B": 1, "Tq": 1, "Tk": 10376, "heads": 16, "kv_heads": 16, "D": 64,
         "t": "f16", "left": 5187, "right": 0, "sinks": 1297, "ragged": False, "packed": False},
        # a batch of single tokens over long caches of different lengths, shared key heads
        {"name": "attn_tokens_batch", "op": "attn", "B": 32, "Tq": 1, "Tk": 16384, "heads": 32, "kv_heads": 8, "D": 128,
         "t": "bf16", "left": 4095, "right": 0, "sinks": 4, "ragged": True, "packed": False},
        # a new view of 1297 tokens over 8 views: bidirectional inside the view (right < 0),
        # back over three views, and the first (reference) view always
        {"name": "attn_new_view", "op": "attn", "B": 1, "Tq": 1297, "Tk": 10376, "heads": 16, "kv_heads": 16, "D": 64,
         "t": "f16", "left": 5187, "right": -1, "sinks": 1297, "ragged": False, "packed": False},
        # two long causal prompts with a short window and shared key heads
        {"name": "attn_prompt", "op": "attn", "B": 2, "Tq": 8192, "Tk": 8192, "heads": 16, "kv_heads": 4, "D": 128,
         "t": "bf16", "left": 1023, "right": 0, "sinks": 4, "ragged": False, "packed": False},
        # a padded batch of odd lengths (one of them empty) out of a packed q | k | v buffer
        {"name": "attn_ragged", "op": "attn", "B": 6, "Tq": 1501, "Tk": 1501, "heads": 12, "kv_heads": 12, "D": 64,
         "t": "f16", "left": 255, "right": 0, "sinks": 5, "ragged": True, "packed": True},
    ]


def _spread(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["linear", "linear", "mlp", "attn", "attn", "attn"])
    if op == "linear":
        K, N = _spread(rng, 64, 4096), _spread(rng, 16, 4096)
        if rng.random() < 0.5:
            K, N = -(-K // 128) * 128, -(-N // 64) * 64
        M = min(_spread(rng, 1, 30000), 350_000_000_000 // (K * N))
        return {"op": op, "M": M, "K": K, "N": N, "x": rng.choice(["f16", "bf16"]),
                "act": rng.choice(["none", "relu", "gelu"]), "out": rng.choice(["f16", "bf16"])}
    if op == "mlp":
        D = rng.choice([384, 768, 1024, _spread(rng, 100, 1500)])
        return {"op": op, "M": _spread(rng, 1, 12000), "D": D, "H": 4 * D}
    D = rng.choice([64, 128])
    kvh = rng.choice([1, 2, 4, 6])
    heads = kvh * rng.choice([1, 1, 2, 3, 4])
    t = rng.choice(["f16", "bf16"])
    if rng.random() < 0.4:  # single tokens, or a few
        Tk = _spread(rng, 1, 30000)
        return {"op": op, "B": _spread(rng, 1, 24), "Tq": rng.choice([1, 1, 1, 2, 5]), "Tk": Tk, "heads": heads,
                "kv_heads": kvh, "D": D, "t": t, "left": rng.choice([-1, _spread(rng, 1, 8192)]), "right": 0,
                "sinks": rng.choice([0, 1, 4, 100]), "ragged": rng.random() < 0.5, "packed": False}
    Tk = _spread(rng, 16, 6000)
    Tq = Tk if rng.random() < 0.6 else max(1, Tk // rng.choice([2, 3, 7]))
    return {"op": op, "B": rng.choice([1, 1, 2, 3]), "Tq": Tq, "Tk": Tk, "heads": heads, "kv_heads": kvh, "D": D, "t": t,
            "left": rng.choice([-1, _spread(rng, 1, 4096), _spread(rng, 1, 4096)]), "right": rng.choice([0, 0, -1, 17]),
            "sinks": rng.choice([0, 1, 4, 64, 300]), "ragged": rng.random() < 0.4, "packed": False}


# ---------------------------------------------------------------------------- e4m3 with scales
def _kb(K):
    return -(-K // 128)


def _quant(x):
    """x [R][K] -> (values of the e4m3 codes in f32 [R][K], exponents e [R][ceil(K/128)] as
    int32): e is the smallest integer with max|x| <= 448 * 2^e over the row's 128 columns (0
    where they are all zero), the codes are x * 2^-e rounded to the nearest e4m3."""
    R, K = x.shape
    nb = _kb(K)
    xf = x.float()
    if nb * 128 != K:
        xf = torch.nn.functional.pad(xf, (0, nb * 128 - K))
    b = xf.view(R, nb, 128)
    amax = b.abs().amax(2)
    m, k = torch.frexp(amax)                      # amax = m * 2^k, m in [0.5, 1)
    e = torch.where(m <= 0.875, k - 9, k - 8)     # 448 = 0.875 * 2^9
    e = torch.where(amax > 0, e, torch.zeros_like(e)).clamp(min=-127)
    codes = torch.ldexp(b, -e[:, :, None]).to(torch.float8_e4m3fn)
    return codes, e


def _scale_tiles(e, K):
    """Exponents [R][nb] -> the scale tiles of include/da3b.h (uint8): [ceil(K/512)]
    [ceil(R/128)][32][4][4], the byte e + 127 of row 128 t + 32 c + l and block 4 g + j at
    [g][t][l][c][j]."""
    R, nb = e.shape
    g, t = -(-K // 512), -(-R // 128)
    full = torch.zeros(t * 128, g * 4, dtype=torch.uint8, device=e.device)
    full[:R, :nb] = (e + 127).to(torch.uint8)
    return full.view(t, 4, 32, g, 4).permute(3, 0, 2, 1, 4).contiguous()


def _tile_scales(tiles, R, nb, dtype=torch.float32):
    """Scale tiles -> scales 2^e [R][nb]."""
    g, t = tiles.shape[:2]
    e = tiles.permute(1, 3, 2, 0, 4).reshape(t * 128, g * 4)[:R, :nb].to(torch.int32) - 127
    return torch.ldexp(torch.ones((), dtype=dtype, device=e.device), e)


def _values(codes, scales, K):
    """Codes [R][nb][128] (or [R][ld]) and scales [R][nb] -> the values [R][K] they stand for."""
    R, nb = scales.shape
    if codes.dim() == 2:
        c = codes[:, :K].to(scales.dtype)
        if nb * 128 != K:
            c = torch.nn.functional.pad(c, (0, nb * 128 - K))
        codes = c.view(R, nb, 128)
    return (codes.to(scales.dtype) * scales[:, :, None]).reshape(R, nb * 128)[:, :K]


def _weights(g, N, K):
    """Weights as a checkpoint holds them: e4m3 codes [N][ld] (ld = K rounded up to 16) and
    scale tiles."""
    w = torch.randn(N, K, device="cuda", generator=g) / math.sqrt(K)
    w = w * torch.exp(0.5 * torch.randn(N, 1, device="cuda", generator=g))
    codes, e = _quant(w)
    ld = -(-K // 16) * 16
    q = torch.zeros(N, ld, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn)
    q.view(torch.uint8)[:, :K] = codes.view(torch.uint8).reshape(N, -1)[:, :K]
    return q, _scale_tiles(e, K)


def _act(y, act):
    if act == "relu":
        return torch.relu(y)
    if act == "gelu":
        return 0.5 * y * (1 + torch.erf(y * math.sqrt(0.5)))
    return y


# ---------------------------------------------------------------------------- attention masks
def _lens(c):
    """Lengths (queries, keys) of each sequence of a case."""
    B, Tq, Tk = c["B"], c["Tq"], c["Tk"]
    if not c["ragged"]:
        return [Tq] * B, [Tk] * B
    kl = [int(Tk * ((0.618034 * i + 0.999) % 1.0)) for i in range(B)]
    if B > 3:
        kl[B // 2] = 0
    return [min(Tq, n) for n in kl], kl


def _visible_pairs(c):
    total = 0
    keys = 0
    for ql, kl in zip(*_lens(c)):
        if ql <= 0 or kl <= 0:
            continue
        p = torch.arange(ql, dtype=torch.float64) + (kl - ql)
        hi = torch.clamp(p + c["right"], max=kl - 1) if c["right"] >= 0 else torch.full_like(p, kl - 1)
        lo = torch.clamp(p - c["left"], min=0) if c["left"] >= 0 else torch.zeros_like(p)
        inside = torch.clamp(hi - lo + 1, min=0)
        front = torch.clamp(torch.minimum(lo, hi + 1), max=c["sinks"])
        total += float((inside + front).sum())
        lo0, hi0 = float(lo.min()), float(hi.max())
        keys += max(0.0, hi0 - lo0 + 1) + min(lo0, c["sinks"])
    return total, keys


def _mask(c, ql, kl, rows):
    """[rows][Tk] truth values: whether the query of row i sees key j, for device lengths
    (ql, kl) of one sequence each [B, 1, 1]."""
    i = rows[None, :, None]
    j = torch.arange(c["Tk"], device=rows.device)[None, None, :]
    p = kl - ql + i
    see = (j < kl) & (i < ql)
    if c["right"] >= 0:
        see = see & (j <= p + c["right"])
    if c["left"] >= 0:
        see = see & ((j >= p - c["left"]) | (j < c["sinks"]))
    return see


# ---------------------------------------------------------------------------- prepare
def prepare(case, seed):
    c = dict(case)
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    s = {"c": c}

    def randn(*shape, dtype=torch.float32):
        return torch.randn(*shape, device="cuda", generator=g, dtype=dtype)

    if c["op"] == "linear":
        M, K, N = c["M"], c["K"], c["N"]
        # activations of transformer layers: a few columns are ten times the others
        x = randn(M, K)
        x = x * torch.where(torch.rand(K, device="cuda", generator=g) < 0.01, 10.0, 1.0)
        s["x"] = x.to(_DT[c["x"]])
        s["w"], s["ws"] = _weights(g, N, K)
        s["bias"] = 0.1 * randn(N)
        if c["out"] == "resid":
            s["resid"] = randn(M, N)
            s["scale"] = 0.1 * (1 + 0.02 * randn(N))  # LayerScale
    elif c["op"] == "mlp":
        M, D, H = c["M"], c["D"], c["H"]
        s["x"] = randn(M, D) * 2 + 0.3
        s["g"] = 1 + 0.1 * randn(D)
        s["b"] = 0.1 * randn(D)
        s["w1"], s["ws1"] = _weights(g, H, D)
        s["w2"], s["ws2"] = _weights(g, D, H)
        s["b1"], s["b2"] = 0.1 * randn(H), 0.1 * randn(D)
    else:
        B, Tq, Tk, h, kvh, D = c["B"], c["Tq"], c["Tk"], c["heads"], c["kv_heads"], c["D"]
        t = _DT[c["t"]]
        if c["packed"]:
            qkv = randn(B, Tk, 3, h, D, dtype=t)
            s["q"], s["k"], s["v"] = qkv[:, :, 0], qkv[:, :, 1], qkv[:, :, 2]
        else:
            s["q"], s["k"], s["v"] = randn(B, Tq, h, D, dtype=t), randn(B, Tk, kvh, D, dtype=t), randn(B, Tk, kvh, D, dtype=t)
        s["q"].mul_(1.5)
        ql, kl = _lens(c)
        s["ql"] = torch.tensor(ql, dtype=torch.int32, device="cuda")
        s["kl"] = torch.tensor(kl, dtype=torch.int32, device="cuda")
    return s


# ---------------------------------------------------------------------------- run
def run(s):
    op = s["c"]["op"]
    if own:
        return _own_linear(s) if op == "linear" else _own_mlp(s) if op == "mlp" else _own_attn(s)
    return _plain_linear(s) if op == "linear" else _plain_mlp(s) if op == "mlp" else _plain_attn(s)


def _product(codes, e, K, w, ws, N):
    """x w^T in f32 of quantised rows (codes, exponents) and held weights."""
    x = _values(codes, torch.ldexp(torch.ones((), device=e.device), e), K)
    return x @ _values(w, _tile_scales(ws, N, _kb(K)), K).t()


def _plain_linear(s):
    c = s["c"]
    codes, e = _quant(s["x"])
    y = _product(codes, e, c["K"], s["w"], s["ws"], c["N"]) + s["bias"]
    if c["out"] == "resid":
        return s["resid"].add_(s["scale"] * y)
    return _act(y, c["act"]).to(_DT[c["out"]])


def _layernorm64(s):
    """LayerNorm in 64 bits (its result is rounded to e4m3, where a value next to a border
    would go either way), in f32."""
    x = s["x"].double()
    d = x - x.mean(1, keepdim=True)
    return (d * torch.rsqrt((d * d).mean(1, keepdim=True) + EPS) * s["g"].double() + s["b"].double()).float()


def _plain_mlp(s):
    c = s["c"]
    codes, e = _quant(_layernorm64(s))
    h = _act(_product(codes, e, c["D"], s["w1"], s["ws1"], c["H"]) + s["b1"], "gelu")
    codes, e = _quant(h)
    return (_product(codes, e, c["H"], s["w2"], s["ws2"], c["D"]) + s["b2"]).half()


def _plain_attn(s):
    c = s["c"]
    B, Tq, h, kvh, D = c["B"], c["Tq"], c["heads"], c["kv_heads"], c["D"]
    r = h // kvh
    q = s["q"].float().view(B, -1, kvh, r, D)[:, :Tq].permute(0, 2, 3, 1, 4)       # B kvh r Tq D
    k = s["k"].float().permute(0, 2, 3, 1)[:, :, None]                              # B kvh 1 D Tk
    v = s["v"].float().permute(0, 2, 1, 3)[:, :, None]                              # B kvh 1 Tk D
    see = _mask(c, s["ql"][:, None, None], s["kl"][:, None, None], torch.arange(Tq, device=q.device))[:, None, None]
    a = torch.matmul(q, k).mul_(1 / math.sqrt(D)).masked_fill_(~see, float("-inf"))
    top = a.amax(-1, keepdim=True)
    p = a.sub_(torch.where(torch.isinf(top), torch.zeros_like(top), top)).exp_()
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p, v) / torch.where(total > 0, total, torch.ones_like(total))
    return o.permute(0, 3, 1, 2, 4).reshape(B, Tq, h, D).to(_DT[c["t"]])


# The library's calls: device pointers, sizes and the current stream.
def _lib():
    from da3cpplib_b200 import _lib as binding

    return binding.load(), torch.cuda.current_stream().cuda_stream


def _ok(rc):
    if rc != 0:
        raise RuntimeError("libda3b returned %d" % rc)


def _own_linear(s):
    c = s["c"]
    lib, st = _lib()
    x, w, M, K, N = s["x"], s["w"], c["M"], c["K"], c["N"]
    ld = w.shape[1]
    xq = torch.empty(M, ld, dtype=torch.uint8, device="cuda")
    xs = torch.empty(lib.da3b_fp8_scale_bytes(M, K), dtype=torch.uint8, device="cuda")
    _ok(lib.da3b_quantize_fp8(x.data_ptr(), _CODE[c["x"]], M, K, K, xq.data_ptr(), ld, xs.data_ptr(), st))
    if c["out"] == "resid":
        r = s["resid"]
        _ok(lib.da3b_linear_fp8_resid_f32(xq.data_ptr(), M, K, ld, xs.data_ptr(), w.data_ptr(), N, ld, s["ws"].data_ptr(),
                                          s["bias"].data_ptr(), s["scale"].data_ptr(), r.data_ptr(), N, st))
        return r
    y = torch.empty(M, N, dtype=_DT[c["out"]], device="cuda")
    _ok(lib.da3b_linear_fp8(xq.data_ptr(), M, K, ld, xs.data_ptr(), w.data_ptr(), N, ld, s["ws"].data_ptr(),
                            s["bias"].data_ptr(), {"none": 0, "relu": 1, "gelu": 2}[c["act"]], y.data_ptr(), _CODE[c["out"]],
                            N, st))
    return y


def _own_mlp(s):
    c = s["c"]
    lib, st = _lib()
    M, D, H = c["M"], c["D"], c["H"]
    ld1, ld2 = s["w1"].shape[1], s["w2"].shape[1]
    xq = torch.empty(M, ld1, dtype=torch.uint8, device="cuda")
    xs = torch.empty(lib.da3b_fp8_scale_bytes(M, D), dtype=torch.uint8, device="cuda")
    hq = torch.empty(M, ld2, dtype=torch.uint8, device="cuda")
    hs = torch.empty(lib.da3b_fp8_scale_bytes(M, H), dtype=torch.uint8, device="cuda")
    y = torch.empty(M, D, dtype=torch.float16, device="cuda")
    _ok(lib.da3b_layernorm_fp8(s["x"].data_ptr(), M, D, D, s["g"].data_ptr(), s["b"].data_ptr(), EPS, xq.data_ptr(), ld1,
                               xs.data_ptr(), st))
    _ok(lib.da3b_linear_fp8_q(xq.data_ptr(), M, D, ld1, xs.data_ptr(), s["w1"].data_ptr(), H, ld1, s["ws1"].data_ptr(),
                              s["b1"].data_ptr(), 2, hq.data_ptr(), ld2, hs.data_ptr(), st))
    _ok(lib.da3b_linear_fp8(hq.data_ptr(), M, H, ld2, hs.data_ptr(), s["w2"].data_ptr(), D, ld2, s["ws2"].data_ptr(),
                            s["b2"].data_ptr(), 0, y.data_ptr(), 0, D, st))
    return y


def _strides(t):
    return (ctypes.c_int64 * 3)(t.stride(0), t.stride(1), t.stride(2))


def _own_attn(s):
    c = s["c"]
    lib, st = _lib()
    q, k, v = s["q"], s["k"], s["v"]
    o = (torch.zeros if c["ragged"] else torch.empty)(c["B"], c["Tq"], c["heads"], c["D"], dtype=q.dtype, device="cuda")
    _ok(lib.da3b_attention_window(q.data_ptr(), _strides(q), k.data_ptr(), _strides(k), v.data_ptr(), _strides(v),
                                  o.data_ptr(), _strides(o), _CODE[c["t"]], c["B"], c["Tq"], c["Tk"], c["heads"],
                                  c["kv_heads"], c["D"], s["ql"].data_ptr() if c["ragged"] else None,
                                  s["kl"].data_ptr() if c["ragged"] else None, c["left"], c["right"], c["sinks"],
                                  1 / math.sqrt(c["D"]), st))
    return o


# ---------------------------------------------------------------------------- work and exact values
def work(case):
    c = dict(case)
    if c["op"] == "linear":
        M, K, N = c["M"], c["K"], c["N"]
        out = 8 if c["out"] == "resid" else 2  # the residual is read and written
        return {"bytes": 2 * M * K + N * K + N * _kb(K) + 4 * N + out * M * N, "flops": 2 * M * N * K}
    if c["op"] == "mlp":
        M, D, H = c["M"], c["D"], c["H"]
        return {"bytes": 4 * M * D + 2 * D * H + 2 * M * D + 4 * (3 * D + H), "flops": 4 * M * D * H}
    pairs, keys = _visible_pairs(c)
    rows = sum(_lens(c)[0])
    return {"bytes": 4 * rows * c["heads"] * c["D"] + 4 * keys * c["kv_heads"] * c["D"] + 8 * c["B"],
            "flops": 4 * pairs * c["heads"] * c["D"]}


def _exact_quant(x):
    """The values [R][K] (64 bits) that x [R][K] stands for once quantised: e4m3 grid points
    by arithmetic (3 mantissa bits, exponents from -6, ties to even)."""
    x = x.double()
    parts = []
    for blk in x.split(128, dim=1):
        amax = blk.abs().amax(1, keepdim=True)
        e = torch.ceil(torch.log2(torch.where(amax > 0, amax, torch.full_like(amax, 448.0)) / 448.0))
        e = torch.where(amax > 448.0 * torch.exp2(e), e + 1, e)
        e = torch.where(amax <= 448.0 * torch.exp2(e - 1), torch.where(amax > 0, e - 1, e), e).clamp(min=-127)
        y = blk * torch.exp2(-e)
        step = torch.exp2(torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6))) - 3)
        parts.append(torch.round(y / step) * step * torch.exp2(e))
    return torch.cat(parts, 1)


def _exact_weight(q, tiles, K):
    N = q.shape[0]
    return _values(q, _tile_scales(tiles, N, _kb(K), torch.float64), K)


def _rows64(x, w, b, act):
    out = []
    for part in x.split(16384):
        out.append(_act(part @ w.t() + b.double(), act))
    return torch.cat(out)


def exact(case, seed):
    s = prepare(case, seed)
    c = s["c"]
    if c["op"] == "linear":
        w = _exact_weight(s["w"], s["ws"], c["K"])
        y = _rows64(_exact_quant(s["x"]), w, s["bias"], c["act"])
        return s["resid"].double() + s["scale"].double() * y if c["out"] == "resid" else y
    if c["op"] == "mlp":
        x = s["x"].double()
        var, mean = torch.var_mean(x, 1, correction=0, keepdim=True)
        n = (x - mean) / torch.sqrt(var + EPS) * s["g"].double() + s["b"].double()
        h = _rows64(_exact_quant(n), _exact_weight(s["w1"], s["ws1"], c["D"]), s["b1"], "gelu")
        return _rows64(_exact_quant(h), _exact_weight(s["w2"], s["ws2"], c["H"]), s["b2"], "none")
    B, Tq, h, kvh, D = c["B"], c["Tq"], c["heads"], c["kv_heads"], c["D"]
    out = torch.zeros(B, Tq, h, D, dtype=torch.float64, device="cuda")
    for b, (ql, kl) in enumerate(zip(*_lens(c))):
        if ql <= 0 or kl <= 0:
            continue
        for r0 in range(0, ql, 2048):
            rows = torch.arange(r0, min(ql, r0 + 2048), device="cuda")
            p = rows + (kl - ql)
            hi = torch.clamp(p + c["right"], max=kl - 1) if c["right"] >= 0 else torch.full_like(p, kl - 1)
            lo = p - c["left"] if c["left"] >= 0 else torch.zeros_like(p)
            j = torch.arange(kl, device="cuda")
            hide = (j[None] > hi[:, None]) | ((j[None] < lo[:, None]) & (j[None] >= c["sinks"]))
            for i in range(h):
                kk, vv = s["k"][b, :kl, i * kvh // h].double(), s["v"][b, :kl, i * kvh // h].double()
                a = (s["q"][b, rows, i].double() @ kk.t()) / math.sqrt(D)
                a = torch.softmax(a.masked_fill(hide, -math.inf), -1)
                out[b, rows, i] = torch.nan_to_num(a, nan=0.0) @ vv
    return out
