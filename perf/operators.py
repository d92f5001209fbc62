"""The operators around the 4-bit linear layers of a training step, as cases to measure: rotary positions, the 8-bit block-scaled
linear layer with its quantizers, and the global gradient norm with clipping.

`own` False: elementary torch operations in 32 bits (64 for angles and norms), rounded once at the end.  `own` True: the calls a
user makes of this package."""
import math

import torch

own = False

F8 = {"e4m3": torch.float8_e4m3fn, "e5m2": torch.float8_e5m2}
F8_MAX = {"e4m3": 448.0, "e5m2": 57344.0}
DTYPE = {"bf16": torch.bfloat16, "f32": torch.float32}


def listed():
    return [
        # positions of one new token of each sequence, far into long contexts
        {"name": "rotary_decode", "op": "rotary", "batch": 8, "t": 1, "hq": 32, "hk": 8, "d": 128, "rot": 128, "interleaved": False,
         "head_major": False, "scale": 1.0, "dtype": "bf16", "max_pos": 131072},
        # a prompt in fp32, two thirds of the head rotated, head-major views, a scaled context's factor, an odd length
        {"name": "rotary_prompt_part", "op": "rotary", "batch": 2, "t": 4097, "hq": 12, "hk": 4, "d": 96, "rot": 64, "interleaved": True,
         "head_major": True, "scale": 1.2079441, "dtype": "f32", "max_pos": 32768},
        # the 30M training configuration: 64 sequences of 512 tokens, 5 heads of 128, packed qkv, forward and backward
        {"name": "rotary_qkv_train", "op": "rotary_qkv", "batch": 64, "t": 512, "hq": 5, "hk": 5, "d": 128, "rot": 128, "interleaved": True,
         "scale": 1.0, "dtype": "bf16"},
        # grouped heads, small heads, an odd length, fp32 (no autocast)
        {"name": "rotary_qkv_grouped", "op": "rotary_qkv", "batch": 3, "t": 1021, "hq": 8, "hk": 2, "d": 64, "rot": 64, "interleaved": False,
         "scale": 1.0, "dtype": "f32"},
        # gradients of the 30M model's parameters (6 blocks, width 640, vocabulary 32000), fp32
        {"name": "clip_30m", "op": "clip", "blocks": 6, "width": 640, "hidden": 1792, "vocab": 32000, "odd": 0, "dtype": "f32", "out": "f32", "max_norm": 1.0},
        # a few small tensors of odd sizes, bf16 gradients into fp32 ones
        {"name": "clip_small", "op": "clip", "blocks": 1, "width": 64, "hidden": 176, "vocab": 257, "odd": 3, "dtype": "bf16", "out": "f32", "max_norm": 0.5},
        # an activation in both orientations, as a training layer wants it
        {"name": "quant_activation", "op": "quant", "rows": 16384, "cols": 4096, "square": False, "transpose": True, "dtype": "bf16", "fmt": "e4m3"},
        # the head's fp32 weight in square blocks, with its transpose
        {"name": "quant_weight", "op": "quant", "rows": 32000, "cols": 640, "square": True, "transpose": True, "dtype": "f32", "fmt": "e4m3"},
        # one token through a packed weight
        {"name": "serve_1", "op": "serve", "m": 1, "k": 4096, "n": 12288, "dtype": "bf16"},
        # a prompt of odd length through the packed head
        {"name": "serve_prompt", "op": "serve", "m": 1021, "k": 640, "n": 32000, "dtype": "bf16"},
        # the head of the 30M model in training, fp32 master weight
        {"name": "train_head", "op": "train", "m": 4096, "k": 640, "n": 32000, "x": "bf16", "w": "f32", "fmt": "e4m3"},
        # a 7B layer in training, a ragged batch of tokens, gradients in e5m2
        {"name": "train_7b", "op": "train", "m": 8187, "k": 4096, "n": 11008, "x": "bf16", "w": "bf16", "fmt": "e5m2"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["rotary", "rotary_qkv", "clip", "quant", "serve", "train"])
    if op in ("rotary", "rotary_qkv"):
        d = rng.choice([32, 64, 80, 96, 128, 192, 256])
        rot = rng.choice([d, d, d // 2, d // 4])
        hk = rng.choice([1, 2, 5, 8])
        c = {"op": op, "batch": _log(rng, 1, 64), "hq": hk * rng.choice([1, 2, 4]), "hk": hk, "d": d, "rot": rot, "interleaved": rng.random() < 0.5,
             "scale": rng.choice([1.0, 1.0, round(rng.uniform(1.0, 1.4), 4)]), "dtype": rng.choice(["bf16", "bf16", "f32"])}
        most = max(1, (60 << 20) // (c["batch"] * (c["hq"] + 2 * hk) * d))
        c["t"] = _log(rng, 1, min(most, 32768))
        if op == "rotary":
            c["head_major"] = rng.random() < 0.5
            c["max_pos"] = rng.choice([4096, 131072, 1 << 20])
        return c
    if op == "clip":
        width = rng.choice([64, 100, 250, 640, 1024])
        return {"op": op, "blocks": rng.choice([1, 2, 6]), "width": width, "hidden": width * 3 - rng.choice([0, 16]), "vocab": _log(rng, 100, 32000),
                "odd": rng.choice([0, 1, 3, 8]), "dtype": rng.choice(["bf16", "f32"]), "out": rng.choice(["f32", "same"]), "max_norm": rng.choice([0.1, 1.0, 1e6])}
    if op == "quant":
        cols = _log(rng, 100, 14336)
        return {"op": op, "rows": _log(rng, 1, min(32768, (64 << 20) // cols)), "cols": cols, "square": rng.random() < 0.4, "transpose": rng.random() < 0.6,
                "dtype": rng.choice(["bf16", "f32"]), "fmt": rng.choice(["e4m3", "e4m3", "e5m2"])}
    if op == "serve":
        k = rng.choice([_log(rng, 200, 11008), 128 * _log(rng, 2, 86)])
        return {"op": op, "m": rng.choice([_log(rng, 1, 128), _log(rng, 1, 4096)]), "k": k, "n": rng.choice([_log(rng, 200, 32000), 128 * _log(rng, 2, 250)]),
                "dtype": rng.choice(["bf16", "bf16", "f32"])}
    return {"op": op, "m": _log(rng, 1, 8192), "k": rng.choice([_log(rng, 200, 4096), 128 * _log(rng, 2, 32)]),
            "n": rng.choice([_log(rng, 200, 11008), 128 * _log(rng, 2, 86)]), "x": rng.choice(["bf16", "bf16", "f32"]), "w": rng.choice(["bf16", "f32"]),
            "fmt": rng.choice(["e4m3", "e5m2"])}


def _clip_shapes(c):
    w, h = c["width"], c["hidden"]
    block = [(w,), (3 * w, w), (w, w), (w,), (2 * h, w), (w, h)]
    return [(c["vocab"], w)] + block * c["blocks"] + [(w,), (c["vocab"], w)] + [(2 * i + 1,) for i in range(c["odd"])]


def _randn(gen, shape, dtype, scale=1.0):
    return (torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32) * scale).to(dtype)


def _activation(gen, rows, cols, dtype):
    """Gaussian rows of differing size with a few columns that stand out, as a residual stream has them."""
    x = torch.randn((rows, cols), generator=gen, device="cuda")
    x = x * torch.exp(0.5 * torch.randn((rows, 1), generator=gen, device="cuda"))
    x[:, :: 97] *= 8.0
    return x.to(dtype)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed) * 1000003 + 17)
    c, s = dict(case), {"case": dict(case)}
    op = c["op"]
    if op in ("rotary", "rotary_qkv"):
        dt, b, t, d = DTYPE[c["dtype"]], c["batch"], c["t"], c["d"]
        s["inv_freq"] = 1.0 / 10000.0 ** (torch.arange(0, c["rot"], 2, device="cuda", dtype=torch.float64) / c["rot"])
        if op == "rotary":
            shape = (lambda h: (b, h, t, d)) if c["head_major"] else (lambda h: (b, t, h, d))
            q, k = _randn(gen, shape(c["hq"]), dt), _randn(gen, shape(c["hk"]), dt)
            s["q"], s["k"] = (q.transpose(1, 2), k.transpose(1, 2)) if c["head_major"] else (q, k)  # [batch, t, heads, d]
            start = torch.randint(0, max(1, c["max_pos"] - t), (b, 1), generator=gen, device="cuda")
            s["pos"] = start + torch.arange(t, device="cuda")
        else:
            s["qkv"] = _randn(gen, (b, t, (c["hq"] + 2 * c["hk"]) * d), dt).requires_grad_()
            s["grads"] = [_randn(gen, (b, h, t, d), dt, 1e-3) for h in (c["hq"], c["hk"], c["hk"])]
    elif op == "clip":
        dt = DTYPE[c["dtype"]]
        size = torch.exp(torch.randn(len(_clip_shapes(c)), generator=gen, device="cuda"))
        s["grads"] = [(torch.randn(sh, generator=gen, device="cuda") * (1e-3 * size[i])).to(dt) for i, sh in enumerate(_clip_shapes(c))]
        s["outs"] = [torch.empty_like(g, dtype=torch.float32 if c["out"] == "f32" else dt) for g in s["grads"]]
    elif op == "quant":
        if c["square"]:
            s["x"] = _randn(gen, (c["rows"], c["cols"]), DTYPE[c["dtype"]], 0.02)
        else:
            s["x"] = _activation(gen, c["rows"], c["cols"], DTYPE[c["dtype"]])
    elif op == "serve":
        s["x"] = _activation(gen, c["m"], c["k"], DTYPE[c["dtype"]])
        s["w"], s["w_sf"] = _quantize(_randn(gen, (c["n"], c["k"]), torch.float32, 0.02), True, "e4m3")[:2]
    else:
        s["x"] = _activation(gen, c["m"], c["k"], DTYPE[c["x"]]).requires_grad_()
        s["w"] = _randn(gen, (c["n"], c["k"]), DTYPE[c["w"]], 0.02).requires_grad_()
        s["e"] = _randn(gen, (c["m"], c["n"]), DTYPE[c["x"]], 1e-3)
    return s


# ---------------------------------------------------------------------------------------------------------------
# plain forms
# ---------------------------------------------------------------------------------------------------------------
def _pad128(t, rows):
    return torch.nn.functional.pad(t, (0, -t.shape[1] % 128, 0, -t.shape[0] % 128 if rows else 0))


def _blocked(e, rows, cols):
    """Scale bytes [rows, cols / 128], one for each block, as the block-scaled product reads them: four equal bytes to a block
    of 128 values, 128 rows by 4 bytes in 512, zeros where no row is."""
    full = torch.zeros(-rows % 128 + rows, cols // 128, dtype=torch.uint8, device=e.device)
    full[:rows] = e
    return full.reshape(-1, 4, 32, cols // 128).permute(0, 3, 2, 1)[..., None].expand(-1, -1, -1, -1, 4).reshape(-1)


def _two(e):
    """2^e as a double for whole e, exactly (a device's exp2 may be off in the last place)."""
    return ((e.to(torch.int64) + 1023) << 52).view(torch.float64)


def _scale_exponent(amax, fmt):
    """The least e with amax <= MAX 2^e (e >= -127)."""
    a = amax.double() / F8_MAX[fmt]
    e = torch.ceil(torch.log2(a.clamp_min(2.0 ** -200)))
    e = torch.where(_two(e - 1) >= a, e - 1, e)
    e = torch.where(_two(e) < a, e + 1, e)
    return e.clamp_min(-127.0)


def _quantize(x, square, fmt):
    """Codes [rows, cols padded to 128], scale bytes, and the exponents [rows, blocks]."""
    rows, cols = x.shape
    v = _pad128(x.detach().float(), square)
    blocks = v.reshape(-1, 128 if square else 1, v.shape[1] // 128, 128)
    e = _scale_exponent(blocks.abs().amax((1, 3)), fmt)
    q = (blocks.double() * _two(-e)[:, None, :, None]).float().to(F8[fmt]).reshape(v.shape)[:rows]
    e = e.repeat_interleave(128, 0)[:rows] if square else e
    return q, _blocked((e + 127).to(torch.uint8), rows, v.shape[1]), e


def _values(q, e, cols):
    return (q.float().reshape(q.shape[0], -1, 128) * _two(e).float()[:, :, None]).reshape(q.shape)[:, :cols]


def _fake(x, square, fmt):
    q, _, e = _quantize(x, square, fmt)
    return _values(q, e, x.shape[1])


def _unblocked(sf, rows, cols):
    kb = -(-cols // 128)
    return sf.reshape(-1, kb, 32, 4, 4)[..., 0].permute(0, 3, 2, 1).reshape(-1, kb)[:rows].float() - 127.0


def _angles(pos, inv_freq, scale):
    a = pos.double()[..., None] * inv_freq
    return (a.cos() * scale).float()[..., None, :], (a.sin() * scale).float()[..., None, :]


def _rotate(x, cos, sin, rot, interleaved):
    f = x.float()
    if interleaved:
        a, b = f[..., :rot:2], f[..., 1:rot:2]
        y = torch.stack([a * cos - b * sin, a * sin + b * cos], -1).flatten(-2)
    else:
        a, b = f[..., : rot // 2], f[..., rot // 2: rot]
        y = torch.cat([a * cos - b * sin, a * sin + b * cos], -1)
    return torch.cat([y, f[..., rot:]], -1).to(x.dtype)


def _split_heads(c, qkv):
    b, t, d = c["batch"], c["t"], c["d"]
    q, k, v = qkv.split([c["hq"] * d, c["hk"] * d, c["hk"] * d], -1)
    return [z.reshape(b, t, -1, d) for z in (q, k, v)]


def _plain(s):
    c = s["case"]
    op = c["op"]
    if op == "rotary":
        cos, sin = _angles(s["pos"], s["inv_freq"], c["scale"])
        return [_rotate(s[n], cos, sin, c["rot"], c["interleaved"]) for n in ("q", "k")]
    if op == "rotary_qkv":
        cos, sin = _angles(torch.arange(c["t"], device="cuda"), s["inv_freq"], c["scale"])
        q, k, v = _split_heads(c, s["qkv"].detach())
        outs = [z.transpose(1, 2).contiguous() for z in (_rotate(q, cos, sin, c["rot"], c["interleaved"]), _rotate(k, cos, sin, c["rot"], c["interleaved"]), v)]
        dq, dk, dv = [g.transpose(1, 2) for g in s["grads"]]
        back = [_rotate(dq, cos, -sin, c["rot"], c["interleaved"]), _rotate(dk, cos, -sin, c["rot"], c["interleaved"]), dv]
        return outs + [torch.cat([z.flatten(-2) for z in back], -1)]
    if op == "clip":
        norm = torch.stack([g.double().square().sum() for g in s["grads"]]).sum().sqrt()
        coef = (c["max_norm"] / (norm + 1e-6)).clamp_max(1.0).float()
        return [norm.float()] + [(g.float() * coef).to(o.dtype) for g, o in zip(s["grads"], s["outs"])]
    if op == "quant":
        q, sf, _ = _quantize(s["x"], c["square"], c["fmt"])
        if not c["transpose"]:
            return [q, sf]
        qt, sft, _ = _quantize(s["x"].T, c["square"], c["fmt"])
        return [q, sf, qt, sft]
    if op == "serve":
        w = _values(s["w"], _unblocked(s["w_sf"], c["n"], c["k"]), c["k"])
        return (_fake(s["x"], False, "e4m3") @ w.T).to(s["x"].dtype)
    x, w, e = s["x"].detach(), s["w"].detach(), s["e"]
    wq = _fake(w, True, "e4m3")
    y = _fake(x, False, "e4m3") @ wq.T
    dx = _fake(e, False, c["fmt"]) @ wq
    dw = _fake(e.T, False, c["fmt"]) @ _fake(x.T, False, "e4m3").T
    return [y.to(x.dtype), dx.to(x.dtype), dw.to(w.dtype)]


# ---------------------------------------------------------------------------------------------------------------
# this package's calls
# ---------------------------------------------------------------------------------------------------------------
def _own(s):
    from quartet_b200 import ops
    from quartet_b200.quantization import fp8_linear
    from quartet_b200.rotary import apply_rotary, rotary_qkv

    c = s["case"]
    op = c["op"]
    if op == "rotary":
        return list(apply_rotary(s["q"], s["k"], s["inv_freq"], s["pos"], interleaved=c["interleaved"], scale=c["scale"]))
    if op == "rotary_qkv":
        outs = rotary_qkv(s["qkv"], c["hq"], c["hk"], s["inv_freq"], interleaved=c["interleaved"], scale=c["scale"])
        return [z.detach() for z in outs] + list(torch.autograd.grad(outs, (s["qkv"],), s["grads"]))
    if op == "clip":
        return [ops.clip_grads(s["grads"], c["max_norm"], out=s["outs"])] + s["outs"]
    if op == "quant":
        got = ops.quant_fp8(s["x"], F8[c["fmt"]], square=c["square"], transpose=c["transpose"])
        return list(got) if c["transpose"] else list(got[:2])
    if op == "serve":
        return ops.linear_fp8(s["x"], s["w"], s["w_sf"])
    y = fp8_linear(s["x"], s["w"], grad_dtype=F8[c["fmt"]])
    return [y.detach()] + list(torch.autograd.grad(y, (s["x"], s["w"]), s["e"]))


def run(state):
    return _own(state) if own else _plain(state)


def work(case):
    c, op = case, case["op"]
    if op in ("rotary", "rotary_qkv"):
        es = 2 if c["dtype"] == "bf16" else 4
        tokens = c["batch"] * c["t"]
        if op == "rotary":
            n = tokens * (c["hq"] + c["hk"])
            return {"bytes": 2 * es * n * c["d"] + 8 * tokens + 4 * c["rot"], "flops": 3 * n * c["rot"]}
        return {"bytes": 2 * 2 * es * tokens * (c["hq"] + 2 * c["hk"]) * c["d"] + 4 * c["rot"], "flops": 2 * 3 * tokens * (c["hq"] + c["hk"]) * c["rot"]}
    if op == "clip":
        n = sum(math.prod(sh) for sh in _clip_shapes(c))
        es = 2 if c["dtype"] == "bf16" else 4
        return {"bytes": n * (es + (4 if c["out"] == "f32" else es)), "flops": 3 * n}
    if op == "quant":
        n = c["rows"] * c["cols"]
        return {"bytes": n * ((2 if c["dtype"] == "bf16" else 4) + (2 if c["transpose"] else 1) * (1 + 1 / 32)), "flops": 3 * n}
    m, n, k = c["m"], c["n"], c["k"]
    if op == "serve":
        es = 2 if c["dtype"] == "bf16" else 4
        return {"bytes": n * k * (1 + 1 / 32) + es * m * (n + k), "flops": 2 * m * n * k}
    ex, ew = (2 if c["x"] == "bf16" else 4), (2 if c["w"] == "bf16" else 4)
    return {"bytes": 2 * ex * m * (n + k) + 2 * ew * n * k, "flops": 6 * m * n * k}


# ---------------------------------------------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------------------------------------------
def _power64(e):
    """2^e for whole e in -400 .. 400."""
    return torch.tensor([2.0 ** i for i in range(-400, 401)], dtype=torch.float64, device=e.device)[e.long() + 400]


def _round8(v, fmt):
    """v to the nearest value of the 8-bit format, ties to the even one."""
    low, bits = (-6, 3) if fmt == "e4m3" else (-14, 2)
    _, p = torch.frexp(v)
    step = _power64((p - 1).clamp_min(low) - bits)
    return (torch.round(v / step) * step).clamp(-F8_MAX[fmt], F8_MAX[fmt])


def _blocks64(x, bl, fmt):
    """Codes' values and exponents of x [rows, cols] in blocks of bl rows by 128 columns."""
    rows, cols = x.shape
    r, k = -(-rows // bl), -(-cols // 128)
    v = torch.zeros(r * bl, k * 128, dtype=torch.float64, device=x.device)
    v[:rows, :cols] = x
    v = v.view(r, bl, k, 128)
    m, p = torch.frexp(v.abs().amax((1, 3)))
    top = 9 if fmt == "e4m3" else 16  # MAX = 0.875 * 2^top
    e = torch.where(m <= 0.875, p - top, p - top + 1).clamp_min(-127)
    e = torch.where(m == 0, torch.full_like(e, -127), e).double()
    q = _round8(v / _power64(e)[:, None, :, None], fmt)
    return q.reshape(r * bl, k * 128)[:rows], e.repeat_interleave(bl, 0)[:rows]


def _values64(x, bl, fmt):
    q, e = _blocks64(x, bl, fmt)
    return (q * _power64(e).repeat_interleave(128, 1))[:, : x.shape[1]]


def _turn64(x, pos, inv_freq, sign, c):
    """The rotation as a product of complex numbers."""
    a = sign * pos.double()[..., None, None] * inv_freq
    z = torch.polar(torch.full_like(a, c["scale"]), a)
    y, r = x.double().clone(), c["rot"]
    i, j = (slice(0, r, 2), slice(1, r, 2)) if c["interleaved"] else (slice(0, r // 2), slice(r // 2, r))
    w = torch.complex(y[..., i], y[..., j]) * z
    y[..., i], y[..., j] = w.real, w.imag
    return y


def exact(case, seed):
    s = prepare(case, seed)
    c, op = case, case["op"]
    if op == "rotary":
        return [_turn64(s[n], s["pos"], s["inv_freq"], 1.0, c) for n in ("q", "k")]
    if op == "rotary_qkv":
        pos = torch.arange(c["t"], device="cuda")
        q, k, v = _split_heads(c, s["qkv"].detach())
        outs = [_turn64(q, pos, s["inv_freq"], 1.0, c), _turn64(k, pos, s["inv_freq"], 1.0, c), v.double()]
        g = [x.transpose(1, 2) for x in s["grads"]]
        back = [_turn64(g[0], pos, s["inv_freq"], -1.0, c), _turn64(g[1], pos, s["inv_freq"], -1.0, c), g[2].double()]
        return [z.transpose(1, 2).contiguous() for z in outs] + [torch.cat([z.reshape(c["batch"], c["t"], -1) for z in back], 2)]
    if op == "clip":
        norm = math.sqrt(math.fsum(float(torch.linalg.vector_norm(g.double())) ** 2 for g in s["grads"]))
        coef = min(1.0, c["max_norm"] / (norm + 1e-6))
        return [torch.tensor(norm, dtype=torch.float64)] + [g.double() * coef for g in s["grads"]]
    if op == "quant":
        got = []
        for x in (s["x"], s["x"].T)[: 2 if c["transpose"] else 1]:
            q, e = _blocks64(x, 128 if c["square"] else 1, c["fmt"])
            by = torch.zeros(-(-x.shape[0] // 128), e.shape[1], 32, 4, 4, dtype=torch.uint8, device="cuda")
            r = torch.arange(x.shape[0], device="cuda")
            by[r // 128, :, r % 32, r % 128 // 32, :] = (e + 127).to(torch.uint8)[:, :, None]
            got += [q, by.reshape(-1)]
        return got
    if op == "serve":
        kb = -(-c["k"] // 128)
        r = torch.arange(c["n"], device="cuda")
        e = s["w_sf"].view(-1, kb, 32, 4, 4)[r // 128, :, r % 32, r % 128 // 32, 0].double() - 127
        w = (s["w"].double() * _power64(e).repeat_interleave(128, 1))[:, : c["k"]]
        return _values64(s["x"], 1, "e4m3") @ w.T
    x, w, e = s["x"].detach(), s["w"].detach(), s["e"]
    wq = _values64(w, 128, "e4m3")
    return [_values64(x, 1, "e4m3") @ wq.T, _values64(e, 1, c["fmt"]) @ wq, _values64(e.T, 1, c["fmt"]) @ _values64(x.T, 1, "e4m3").T]
