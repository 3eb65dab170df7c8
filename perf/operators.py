"""Cases that measure the microscaled operators: 4-bit quantisation, its
inverse, products of 4-bit matrices (serving and training) and the gated SiLU
whose inputs are kept in 8 bits for the backward pass.

Formats. A row is cut into blocks of 32 along its last axis (the last block may
be shorter). A block with largest magnitude a = m 2^e (1 <= m < 2) has one scale
2^s, stored as the byte s + 127:
  mxfp4:   s = max(e - 2, -127); values round (ties to even) to
           0, .5, 1, 1.5, 2, 3, 4, 6 times 2^s, at most 6; two codes per byte,
           the lower index in the lower half (bit 3 is the sign).
  mxint8:  s = max(e, -120); values round (ties to even) to k 2^(s - 6),
           |k| <= 127.
A block that holds an infinity or a NaN has scale byte 255 and stands for NaN.
Matrices of codes are row-major, rows padded to whole blocks with zeros. The
scales of an mxfp4 matrix are kept in tiles of 128 rows x 4 blocks, 512 bytes
each, byte 16 (r mod 32) + 4 (r / 32) + b of a tile for row r and block b.
"""
import math

import torch

own = False

BLOCK = 32
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


# ---- the cases ---------------------------------------------------------------

def listed():
    return [
        # serving: one token through an attention output projection of the 7B-shaped model
        {"name": "token 4096x4096", "op": "linear", "m": 1, "n": 4096, "k": 4096, "type": "f16"},
        # serving: a batch of 16 decoding requests through the largest weight of the 70B-shaped model
        {"name": "16 tokens 28672x8192", "op": "linear", "m": 16, "n": 28672, "k": 8192, "type": "bf16"},
        # serving: a prompt of odd length through a gate projection of the 7B-shaped model
        {"name": "prompt 777 11008x4096", "op": "linear", "m": 777, "n": 11008, "k": 4096, "type": "f16"},
        # serving: eight prompts of 1024 tokens through a gate projection of the 70B-shaped model
        {"name": "prompt 8192 28672x8192", "op": "linear", "m": 8192, "n": 28672, "k": 8192, "type": "bf16"},
        # training: output, input gradient and weight gradient of an up projection of the 7B-shaped model
        {"name": "train 2048 11008x4096", "op": "train", "m": 2048, "n": 11008, "k": 4096, "type": "bf16"},
        # training: a key projection of the 70B-shaped model, a batch whose length is no multiple of a block
        {"name": "train 1003 1024x8192", "op": "train", "m": 1003, "n": 1024, "k": 8192, "type": "f16"},
        # activations of one decoded token, quantised and read back
        {"name": "round trip 1x8192", "op": "quantize", "m": 1, "k": 8192, "both": False, "type": "bf16"},
        # activations of eight sequences, quantised along features and along tokens, and read back
        {"name": "round trip 8192x4096 both", "op": "quantize", "m": 8192, "k": 4096, "both": True, "type": "f32"},
        # a fetched weight expanded to the [in, out] layout that a 16-bit product takes
        {"name": "expand 28672x8192 to in,out", "op": "dequantize", "n": 28672, "k": 8192, "transpose": True, "type": "f16"},
        # a small weight of odd extents expanded in its own layout
        {"name": "expand 1001x4100", "op": "dequantize", "n": 1001, "k": 4100, "transpose": False, "type": "f32"},
        # training: the gated SiLU of the 7B-shaped model over eight sequences
        {"name": "gate 8192x11008", "op": "gate", "m": 8192, "k": 11008, "type": "bf16"},
        # training: a short odd batch of a small model
        {"name": "gate 13x1003", "op": "gate", "m": 13, "k": 1003, "type": "f32"},
    ]


def draw(rng):
    def size(lo, hi):
        v = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
        if rng.random() < 0.4:  # whole tiles are as common as odd sizes
            v = v // 64 * 64 or v
        return min(max(v, lo), hi)

    op = rng.choice(["linear", "linear", "linear", "train", "quantize", "dequantize", "gate"])
    kind = rng.choice(["f16", "bf16"])
    any_kind = rng.choice(["f32", "f16", "bf16"])
    if op == "linear":
        return {"op": op, "m": size(1, 8192), "n": size(64, 28672), "k": size(64, 8192), "type": kind}
    if op == "train":
        return {"op": op, "m": size(1, 4096), "n": size(64, 11008), "k": size(64, 8192), "type": kind}
    if op == "quantize":
        return {"op": op, "m": size(1, 8192), "k": size(32, 8192), "both": rng.random() < 0.5, "type": any_kind}
    if op == "dequantize":
        return {"op": op, "n": size(64, 28672), "k": size(64, 8192), "transpose": rng.random() < 0.5, "type": any_kind}
    return {"op": op, "m": size(1, 8192), "k": size(32, 11008), "type": any_kind}


def _padded(k):
    return -(-k // BLOCK) * BLOCK


def _held(rows, k):
    """Bytes of an mxfp4 matrix: codes and scales."""
    return rows * _padded(k) // 2 + rows * _padded(k) // BLOCK


def work(case):
    w = TYPES[case["type"]].itemsize
    op = case["op"]
    if op == "linear":
        m, n, k = case["m"], case["n"], case["k"]
        return {"bytes": m * k * w + _held(n, k) + m * n * w, "flops": 2 * m * n * k}
    if op == "train":  # reads x, w, dy; writes y, dx, dw; three products
        m, n, k = case["m"], case["n"], case["k"]
        return {"bytes": 2 * (m * k + n * k + m * n) * w, "flops": 6 * m * n * k}
    if op == "quantize":
        n = case["m"] * case["k"]
        return {"bytes": n * w * (3 if case["both"] else 2), "flops": n}
    if op == "dequantize":
        return {"bytes": _held(case["n"], case["k"]) + case["n"] * case["k"] * w, "flops": case["n"] * case["k"]}
    n = case["m"] * case["k"]
    # forward: gate, up -> h and two 8-bit copies; backward: dh and the copies -> dgate, dup
    kept = 2 * case["m"] * (_padded(case["k"]) * (BLOCK + 1) // BLOCK)
    return {"bytes": 6 * n * w + 2 * kept, "flops": 20 * n}


# ---- inputs ------------------------------------------------------------------

def _normal(shape, std, dtype, g):
    return torch.empty(shape, device="cuda").normal_(0, std, generator=g).to(dtype)


def _activations(m, k, dtype, g):
    """Normal values with a few loud features, as the residual stream of a model has."""
    x = torch.empty(m, k, device="cuda").normal_(0, 1, generator=g)
    loud = torch.empty(k, device="cuda").uniform_(0, 1, generator=g) < 0.01
    return torch.where(loud, x * 12, x).to(dtype)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    t = TYPES[case["type"]]
    op = case["op"]
    s = {"case": case, "dtype": t}
    if op in ("linear", "dequantize"):  # the weight is held in 4 bits
        weight = _normal((case["n"], case["k"]), 0.02, torch.float32, g)
        s["codes"], s["scales"] = _pack(*_quantize4(weight))
    if op == "linear":
        s["x"] = _activations(case["m"], case["k"], t, g)
    elif op == "train":
        s["x"] = _activations(case["m"], case["k"], t, g).requires_grad_()
        s["weight"] = _normal((case["n"], case["k"]), 0.02, t, g).requires_grad_()
        s["dy"] = _normal((case["m"], case["n"]), 1e-2, t, g)
    elif op == "quantize":
        s["x"] = _activations(case["m"], case["k"], t, g)
    elif op == "gate":
        s["gate"] = _normal((case["m"], case["k"]), 1.5, t, g).requires_grad_()
        s["up"] = _normal((case["m"], case["k"]), 1.0, t, g).requires_grad_()
        s["dh"] = _normal((case["m"], case["k"]), 1e-2, t, g)
    return s


# ---- the plain form ----------------------------------------------------------

def _blocks(x):
    """x [rows, k] in 32 bits, in blocks [rows, blocks, 32]."""
    rows, k = x.shape
    return torch.nn.functional.pad(x.float(), (0, _padded(k) - k)).view(rows, -1, BLOCK)


def _top(b):
    """Per block: the exponent of the largest magnitude, and whether all values are finite."""
    a = b.abs().amax(-1, keepdim=True)
    fine = torch.isfinite(a)
    e = torch.frexp(torch.where(fine, a, torch.ones_like(a)))[1] - 1
    return torch.where(a > 0, e, torch.full_like(e, -1000)), fine


def _scaled(b, power):
    """b 2^power, exactly: two factors, since one may be out of range. Their
    bits are put together, as pow() need not be exact."""
    half = power // 2
    two = [((p + 127).int() << 23).view(torch.float32) for p in (half, power - half)]
    return b * two[0] * two[1]


def _quantize4(x):
    """Codes 0..15 [rows, blocks, 32] and scale bytes [rows, blocks]."""
    b = _blocks(x)
    e, fine = _top(b)
    s = (e - 2).clamp(min=-127)
    v = _scaled(b, -s)
    a = v.abs()
    code = ((a > 0.25).to(torch.uint8) + (a >= 0.75) + (a > 1.25) + (a >= 1.75) + (a > 2.5) + (a >= 3.5) + (a > 5))
    code = torch.where(fine, code | (torch.signbit(b).to(torch.uint8) << 3), 0).to(torch.uint8)
    return code, torch.where(fine, s + 127, 255).to(torch.uint8).squeeze(-1)


def _values4(code, scale):
    """The values that codes [rows, blocks, 32] and scale bytes [rows, blocks] stand for, [rows, 32 blocks] in 32 bits."""
    table = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6, -0.0, -0.5, -1, -1.5, -2, -3, -4, -6], device=code.device)
    s = scale.unsqueeze(-1).int() - 127
    v = _scaled(table[code.int()], s)
    return torch.where(s == 128, torch.full_like(v, math.nan), v).flatten(1)


def _quantize8(x):
    """The values that x stands for once held in mxint8, in 32 bits."""
    b = _blocks(x)
    e, fine = _top(b)
    s = e.clamp(min=-120)
    q = torch.round(_scaled(b, 6 - s)).clamp(-127, 127)
    v = torch.where(fine, _scaled(q, s - 6), torch.full_like(q, math.nan))
    return v.flatten(1)[:, :x.shape[1]]


def _pack(code, scale):
    """Two codes per byte, and the scales in tiles of 128 rows x 4 blocks."""
    rows, blocks = scale.shape
    two = code.view(rows, -1, 2)
    tiles = torch.nn.functional.pad(scale, (0, -blocks % 4, 0, -rows % 128))
    tiles = tiles.view(-(-rows // 128), 4, 32, -(-blocks // 4), 4).permute(0, 3, 2, 1, 4).contiguous()
    return two[..., 0] | (two[..., 1] << 4), tiles.flatten()


def _unpack(codes, scales, rows):
    blocks = codes.shape[1] // 16
    code = torch.stack((codes & 15, codes >> 4), -1).view(rows, blocks, BLOCK)
    tiles = scales.view(-(-rows // 128), -(-blocks // 4), 32, 4, 4).permute(0, 3, 2, 1, 4)
    return code, tiles.reshape(-(-rows // 128) * 128, -1)[:rows, :blocks]


def _round4(x):
    """x [rows, k] as its mxfp4 form stands for it, in 32 bits, rows padded to whole blocks."""
    return _values4(*_quantize4(x))


def _plain(s):
    case, t = s["case"], s["dtype"]
    op = case["op"]
    if op == "linear":
        w = _values4(*_unpack(s["codes"], s["scales"], case["n"]))
        return {"y": (_round4(s["x"]) @ w.t()).to(t)}
    if op == "train":
        x, w, dy = s["x"].detach(), s["weight"].detach(), s["dy"]
        y = _round4(x) @ _round4(w).t()
        dx = _round4(dy) @ _round4(w.t()).t()
        dw = _round4(dy.t()) @ _round4(x.t()).t()
        return {"y": y.to(t), "dx": dx.to(t), "dw": dw.to(t)}
    if op == "quantize":
        k = case["k"]
        out = {"values": _round4(s["x"])[:, :k].to(t)}
        if case["both"]:
            out["across"] = _round4(s["x"].t())[:, :case["m"]].to(t)
        return out
    if op == "dequantize":
        v = _values4(*_unpack(s["codes"], s["scales"], case["n"]))[:, :case["k"]]
        return {"w": (v.t() if case["transpose"] else v).to(t).contiguous()}
    g, u = s["gate"].detach().float(), s["up"].detach().float()
    h = g / (1 + torch.exp(-g)) * u
    g, u, dh = _quantize8(g), _quantize8(u), s["dh"].float()
    sig = 1 / (1 + torch.exp(-g))
    return {"h": h.to(t), "dgate": (dh * u * sig * (1 + g * (1 - sig))).to(t), "dup": (dh * g * sig).to(t)}


# ---- the framework's operators -----------------------------------------------

def _own(s):
    from sym_b200 import microscale as mx

    case, t = s["case"], s["dtype"]
    op = case["op"]
    if op == "linear":
        return {"y": mx.linear(s["x"], mx.MxTensor(s["codes"], s["scales"], (case["n"], case["k"])))}
    if op == "train":
        y = mx.linear(s["x"], s["weight"])
        dx, dw = torch.autograd.grad(y, (s["x"], s["weight"]), s["dy"])
        return {"y": y.detach(), "dx": dx, "dw": dw}
    if op == "quantize":
        if case["both"]:
            q, across = mx.quantize_both(s["x"])
            return {"values": mx.dequantize(q, t), "across": mx.dequantize(across, t)}
        return {"values": mx.dequantize(mx.quantize(s["x"]), t)}
    if op == "dequantize":
        w = mx.MxTensor(s["codes"], s["scales"], (case["n"], case["k"]))
        return {"w": mx.dequantize(w, t, transpose=case["transpose"])}
    h = mx.silu_mul(s["gate"], s["up"])
    dgate, dup = torch.autograd.grad(h, (s["gate"], s["up"]), s["dh"])
    return {"h": h.detach(), "dgate": dgate, "dup": dup}


def run(state):
    return _own(state) if own else _plain(state)


# ---- the definition, in 64 bits ------------------------------------------------

def _two_to(e):
    """2^e in 64 bits for whole numbers e of the normal range."""
    return ((e.long() + 1023) << 52).view(torch.float64)


def _exact_round(x, bits):
    """Rows of x as held in `bits` bits, from the definition: every block is
    divided by its scale and rounded on the grid of its element type."""
    rows, k = x.shape
    out = torch.zeros(rows, _padded(k), dtype=torch.float64, device=x.device)
    out[:, :k] = x.double()
    b = out.view(rows, -1, BLOCK)
    top = b.abs().max(-1, keepdim=True).values
    e = torch.floor(torch.log2(torch.where(torch.isfinite(top), top, 1.0).clamp(min=1e-300)))
    e = torch.where(_two_to(e) > top, e - 1, e)  # log2 may round to a whole number
    e = torch.where(_two_to(e + 1) <= top, e + 1, e)
    if bits == 4:
        scale = _two_to((e - 2).clamp(min=-127.0))
        v = b / scale
        a = v.abs()
        step = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0)).double()
        q = torch.sign(v) * (torch.round(a / step) * step).clamp(max=6.0)
    else:
        scale = _two_to(e.clamp(min=-120.0) - 6)
        q = torch.round(b / scale).clamp(-127, 127)
    v = torch.where(torch.isfinite(top), q * scale, torch.full_like(q, math.nan))
    return v.view(rows, -1)


def _exact_weight(s):
    """The values of the packed weight, read byte by byte from its layout."""
    n, k = s["case"]["n"], s["case"]["k"]
    codes, scales = s["codes"], s["scales"]
    blocks = codes.shape[1] // 16
    cols = torch.arange(k, device=codes.device)
    r = torch.arange(n, device=codes.device).unsqueeze(1)
    nibble = (codes[:, cols // 2].int() >> (4 * (cols % 2))) & 15
    mag = nibble & 7
    value = torch.where(mag < 2, mag * 0.5, _two_to(mag // 2 - 1) * (1 + 0.5 * (mag % 2)))
    value = torch.where(nibble >= 8, -value, value).double()
    at = torch.arange(blocks, device=codes.device)
    byte = ((r // 128) * (-(-blocks // 4)) + at // 4) * 512 + 16 * (r % 32) + 4 * (r % 128 // 32) + at % 4
    scale = _two_to(scales[byte].long() - 127)
    return value * scale.repeat_interleave(BLOCK, 1)[:, :k]


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "linear":
        return {"y": _exact_round(s["x"], 4)[:, :case["k"]] @ _exact_weight(s).t()}
    if op == "train":
        x, w, dy = s["x"].detach(), s["weight"].detach(), s["dy"]
        return {"y": _exact_round(x, 4) @ _exact_round(w, 4).t(),
                "dx": _exact_round(dy, 4) @ _exact_round(w.t(), 4).t(),
                "dw": _exact_round(dy.t(), 4) @ _exact_round(x.t(), 4).t()}
    if op == "quantize":
        out = {"values": _exact_round(s["x"], 4)[:, :case["k"]]}
        if case["both"]:
            out["across"] = _exact_round(s["x"].t(), 4)[:, :case["m"]]
        return out
    if op == "dequantize":
        w = _exact_weight(s)
        return {"w": (w.t() if case["transpose"] else w).contiguous()}
    g, u = s["gate"].detach().double(), s["up"].detach().double()
    h = g * torch.sigmoid(g) * u
    g, u, dh = _exact_round(g, 8)[:, :case["k"]], _exact_round(u, 8)[:, :case["k"]], s["dh"].double()
    sig = torch.sigmoid(g)
    return {"h": h, "dgate": dh * u * (sig + g * sig * torch.sigmoid(-g)), "dup": dh * g * sig}
