"""Measured cases of the microscaled (4- and 8-bit) operators around a LoRA linear.

Four operators, each in its plain form (elementary torch operations in 32 bits, rounded
once at the end) and, where ``own`` is true, as a user calls it in ``probe_b200.mx``:

``quantize``    x -> 4-bit codes with a scale per block (mxfp4: 32 values and a power of
                two; nvfp4: 16 values, an E4M3 scale and one 32-bit scale per tensor), and
                the values that they stand for
``checkpoint``  an activation kept for the backward pass in 8 bits (mxfp8: E4M3 codes, a
                power of two per 32 values), and the values that it stands for
``linear``      y = q(x) W^T + bias + s (x A^T) B^T with W and q(x) in 4 bits, A, B and the
                adapter's x in 16
``backward``    of that linear from the 8-bit checkpoint X of its input and z = s x A^T:
                dA = s (dy B)^T X, dB = dy^T z and, where asked for, dx = dy W + s (dy B) A

Layouts: codes are row-major, two 4-bit codes a byte, the even column in the low half;
rows are padded to whole blocks of 32.  Scales lie in 512-byte chunks of 128 rows by 4
blocks: row r, block g of a chunk at byte 16 (r % 32) + 4 (r / 32) + g.  z is the pair
[hi | lo] in the activations' type, each part round_up(r, 16) wide, zero beyond r.
"""

import math

import torch

own = False

DEV = "cuda"
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
BLOCK = {"mxfp4": 32, "nvfp4": 16, "mxfp8": 32}


# ------------------------------------------------------------------------------- cases
def listed():
    return [
        # one decoding step's activations of a 16-sequence batch
        {"name": "q4 mx 16x4096", "op": "quantize", "fmt": "mxfp4", "m": 16, "k": 4096, "dtype": "bf16"},
        # a feed-forward weight, quantised when a model is loaded
        {"name": "q4 nv 13824x5120", "op": "quantize", "fmt": "nvfp4", "m": 13824, "k": 5120, "dtype": "bf16"},
        # a short, odd training batch
        {"name": "save8 255x4096", "op": "checkpoint", "m": 255, "k": 4096, "dtype": "fp16"},
        # the tokens of one video sample
        {"name": "save8 32760x5120", "op": "checkpoint", "m": 32760, "k": 5120, "dtype": "bf16"},
        # one token through an up projection
        {"name": "linear m1 mx", "op": "linear", "fmt": "mxfp4", "m": 1, "n": 11008, "k": 4096, "r": 16,
         "bias": False, "dtype": "bf16"},
        # a batch of 64 decoding sequences
        {"name": "linear m64 nv", "op": "linear", "fmt": "nvfp4", "m": 64, "n": 11008, "k": 4096, "r": 16,
         "bias": False, "dtype": "bf16"},
        # a short ragged prompt, odd rank, with a bias
        {"name": "linear m333 mx", "op": "linear", "fmt": "mxfp4", "m": 333, "n": 4096, "k": 4096, "r": 20,
         "bias": True, "dtype": "fp16"},
        # a prefill of an odd number of tokens into a feed-forward projection
        {"name": "linear m4095 mx", "op": "linear", "fmt": "mxfp4", "m": 4095, "n": 13824, "k": 5120, "r": 16,
         "bias": True, "dtype": "bf16"},
        # one video sample through an attention projection with three adapters stacked
        {"name": "linear m32760 nv", "op": "linear", "fmt": "nvfp4", "m": 32760, "n": 5120, "k": 5120, "r": 224,
         "bias": False, "dtype": "bf16"},
        # a small training batch
        {"name": "backward m256", "op": "backward", "fmt": "mxfp4", "m": 256, "n": 4096, "k": 4096, "r": 16,
         "dx": True, "dtype": "bf16"},
        # a language model's training step, up projection, gradient passed on
        {"name": "backward m4097", "op": "backward", "fmt": "nvfp4", "m": 4097, "n": 11008, "k": 4096, "r": 16,
         "dx": True, "dtype": "bf16"},
        # the first projection of a video model: the adapters' gradients alone
        {"name": "backward m32760", "op": "backward", "fmt": "mxfp4", "m": 32760, "n": 5120, "k": 5120, "r": 224,
         "dx": False, "dtype": "bf16"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["quantize", "checkpoint", "linear", "linear", "backward", "backward"])
    dtype = rng.choice(["bf16", "bf16", "fp16"])
    if op in ("quantize", "checkpoint"):
        m, k = _log(rng, 1, 32760), _log(rng, 64, 13824)
        while m * k > 32760 * 5120:
            m = max(1, m // 2)
        case = {"op": op, "m": m, "k": k, "dtype": dtype}
        if op == "quantize":
            case["fmt"] = rng.choice(["mxfp4", "nvfp4"])
        return case
    m, k, n = _log(rng, 1, 32760), 32 * _log(rng, 8, 432), _log(rng, 256, 13824)
    if rng.random() < 0.6:
        n = (n + 63) // 64 * 64
    while m * k * n > 32760 * 5120 * 5120:
        m = max(1, m // 2)
    case = {"op": op, "fmt": rng.choice(["mxfp4", "nvfp4"]), "m": m, "n": n, "k": k,
            "r": rng.choice([4, 8, 12, 16, 16, 32, 64, 128, 224]), "dtype": dtype}
    if op == "linear":
        case["bias"] = rng.random() < 0.5
    else:
        case["dx"] = rng.random() < 0.7
    return case


# -------------------------------------------------------------- the formats, in 32 bits
def _pow2(e):
    """2^e for whole e in [-127, 127], exactly."""
    return torch.where(e < -126, torch.full_like(e, 0x00400000), (e + 127) << 23).to(torch.int32).view(torch.float32)


def _round_e2m1(y):
    a = y.abs()
    step = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0))
    return torch.clamp(torch.round(a / step) * step, max=6.0) * torch.sign(y)


def _round_e4m3(y):
    a = torch.clamp(y.abs(), max=448.0)
    e = torch.clamp(((a.view(torch.int32) >> 23) & 255) - 127, min=-6)
    step = _pow2(e - 3)
    return torch.clamp(torch.round(a / step) * step, max=448.0) * torch.sign(y)


def _split(x, fmt):
    """x in 32 bits, padded to whole blocks of 32 columns, and cut into the format's blocks."""
    m, k = x.shape
    p = torch.zeros((m, (k + 31) // 32 * 32), device=x.device, dtype=torch.float32)
    p[:, :k] = x
    return p.view(m, -1, BLOCK[fmt])


def _plain_quantize(x, fmt, g):
    """(values in units of the scale [m, blocks, block], scale [m, blocks, 1]) of the format."""
    b = _split(x, fmt)
    amax = b.abs().amax(dim=2, keepdim=True)
    if fmt == "nvfp4":
        s = _round_e4m3(amax / torch.tensor(6.0 * g, dtype=torch.float32, device=x.device))
        unit = s * g
        q = _round_e2m1(torch.where(unit > 0, b / torch.where(unit > 0, unit, 1.0), 0.0))
        return q, s
    top = 2 if fmt == "mxfp4" else 8
    e = torch.clamp(((amax.view(torch.int32) >> 23) & 255) - 127 - top, min=-127)
    y = b * _pow2(-e)
    return (_round_e2m1(y) if fmt == "mxfp4" else _round_e4m3(y)), _pow2(e)


def _plain_values(x, fmt, g):
    q, s = _plain_quantize(x, fmt, g)
    return (q * s * g).reshape(x.shape[0], -1)[:, :x.shape[1]]


def _codes(q, fmt):
    """Bytes of the codes of values in units of the scale."""
    sign = (q < 0).to(torch.int32)
    a = q.abs()
    if fmt == "mxfp8":
        e = ((a.view(torch.int32) >> 23) & 255) - 127
        low = e < -6
        man = torch.where(low, a * 512.0, (a / _pow2(torch.clamp(e, min=-6)) - 1.0) * 8.0).to(torch.int32)
        return ((sign << 7) | torch.where(low, man, ((e + 7) << 3) | man)).to(torch.uint8).reshape(q.shape[0], -1)
    c = torch.where(a < 2, a * 2, torch.where(a < 4, a + 2, a / 2 + 4)).to(torch.int32) | (sign << 3)
    c = c.reshape(q.shape[0], -1)
    return (c[:, 0::2] | (c[:, 1::2] << 4)).to(torch.uint8)


def _tiled(s, fmt):
    """Bytes of the scales [m, blocks, 1] in chunks of 128 rows by 4 blocks."""
    m, nb, _ = s.shape
    if fmt == "nvfp4":
        code = _codes(s.view(m, nb, 1), "mxfp8").view(m, nb)
    else:
        code = ((s.view(torch.int32) >> 23) & 255).view(m, nb).to(torch.uint8)
    p = torch.zeros(((m + 127) // 128 * 128, (nb + 3) // 4 * 4), device=s.device, dtype=torch.uint8)
    p[:m, :nb] = code
    return p.view(-1, 4, 32, p.shape[1] // 4, 4).permute(0, 3, 2, 1, 4).contiguous().view(-1)


def _untiled(t, m, nb):
    gb = (nb + 3) // 4
    return t.view(-1, gb, 32, 4, 4).permute(0, 3, 2, 1, 4).reshape(-1, gb * 4)[:m, :nb]


def _of_e4m3(c):
    c = c.to(torch.int32)
    e, man = (c >> 3) & 15, (c & 7).float()
    v = torch.where(e == 0, man / 512.0, (1.0 + man / 8.0) * _pow2(torch.clamp(e, min=1) - 7))
    return torch.where(c > 127, -v, v)


def _decode(t):
    """The values, in 32 bits, that codes and scales stand for."""
    m, k = t["shape"]
    fmt = t["fmt"]
    if fmt == "mxfp8":
        q = _of_e4m3(t["codes"])
    else:
        c = torch.stack([t["codes"] & 15, t["codes"] >> 4], dim=2).reshape(m, -1).to(torch.int32)
        a = (c & 7).float()
        a = torch.where(a < 4, a / 2, torch.where(a < 6, a - 2, 2 * a - 8))
        q = torch.where(c > 7, -a, a)
    nb = q.shape[1] // BLOCK[fmt]
    s = _untiled(t["scales"], m, nb)
    s = _of_e4m3(s) if fmt == "nvfp4" else _pow2(s.to(torch.int32) - 127)
    return (q.view(m, nb, -1) * s[:, :, None] * t["global_scale"]).reshape(m, -1)[:, :k]


# ------------------------------------------------------------------------------ inputs
def _f32(v):
    return float(torch.tensor(v, dtype=torch.float32))


def _pack(x, fmt, g=1.0):
    q, s = _plain_quantize(x, fmt, g)
    return {"codes": _codes(q, fmt), "scales": _tiled(s, fmt), "shape": tuple(x.shape), "fmt": fmt,
            "global_scale": g}


def _activations(gen, m, k, dtype):
    """Normal values with some columns several times as wide as the others, as activations are."""
    wide = torch.rand(k, generator=gen, device=DEV) < 0.01
    x = torch.randn(m, k, generator=gen, device=DEV)
    return (x * torch.where(wide, 8.0, 1.0)).to(dtype)


def _global(fmt, amax):
    """The tensor-wide scale that maps amax to the largest value of the format."""
    return _f32(amax / (448.0 * 6.0)) if fmt == "nvfp4" else 1.0


def prepare(case, seed):
    gen = torch.Generator(device=DEV)
    gen.manual_seed(seed)
    dtype = DTYPES[case["dtype"]]
    m, k, op = case["m"], case["k"], case["op"]
    st = {"op": op}
    if op == "checkpoint":
        return {**st, "x": _activations(gen, m, k, dtype), "fmt": "mxfp8", "global_scale": 1.0}
    if op == "quantize":
        # 38.73: about the largest value of such activations, as calibration would give it
        return {**st, "x": _activations(gen, m, k, dtype), "fmt": case["fmt"],
                "global_scale": _global(case["fmt"], 38.73)}
    n, r, fmt = case["n"], case["r"], case["fmt"]
    w = torch.randn(n, k, generator=gen, device=DEV) / math.sqrt(k)
    st["w"] = _pack(w, fmt, _global(fmt, 6.0 / math.sqrt(k)))
    del w
    st["a"] = (torch.randn(r, k, generator=gen, device=DEV) / math.sqrt(k)).to(dtype)
    st["b"] = (torch.randn(n, r, generator=gen, device=DEV) / math.sqrt(r)).to(dtype)
    st["scale"] = 2.0
    x = _activations(gen, m, k, dtype)
    if op == "linear":
        st["bias"] = torch.randn(n, generator=gen, device=DEV).to(dtype) if case["bias"] else None
        st["x"], st["x_global"] = x, _global(fmt, 38.73)
        return st
    st["x8"] = _pack(x, "mxfp8")
    z = (2.0 * (x.float() @ st["a"].float().t())).to(torch.float32)
    r16 = (r + 15) // 16 * 16
    st["z"] = torch.zeros(m, 2 * r16, device=DEV, dtype=dtype)
    st["z"][:, :r] = z.to(dtype)
    st["z"][:, r16:r16 + r] = z - st["z"][:, :r].float()
    st["dy"] = (torch.randn(m, n, generator=gen, device=DEV) / math.sqrt(n)).to(dtype)
    st["dx"] = case["dx"]
    return st


# ------------------------------------------------------------------------------- passes
def _run_own(st):
    from probe_b200 import mx

    def held(t):
        return mx.MXTensor(t["codes"], t["scales"], t["shape"], t["fmt"], t["global_scale"])

    if st["op"] in ("quantize", "checkpoint"):
        q = mx.mx_quantize(st["x"], st["fmt"], global_scale=st["global_scale"])
        return {"values": mx.mx_dequantize(q, dtype=st["x"].dtype)}
    if st["op"] == "linear":
        return {"y": mx.mx_lora_linear(st["x"], held(st["w"]), st["bias"], st["a"], st["b"], st["scale"],
                                       x_global_scale=st["x_global"])}
    dx, da, db = mx.mx_lora_backward(st["dy"], held(st["x8"]), st["z"], st["a"], st["b"], st["scale"],
                                     weight=held(st["w"]) if st["dx"] else None)
    return {"dx": dx, "da": da, "db": db}


def _run_plain(st):
    if st["op"] in ("quantize", "checkpoint"):
        return {"values": _plain_values(st["x"], st["fmt"], st["global_scale"]).to(st["x"].dtype)}
    a, b = st["a"].float(), st["b"].float()
    if st["op"] == "linear":
        x = st["x"].float()
        y = _plain_values(x, st["w"]["fmt"], st["x_global"]) @ _decode(st["w"]).t()
        y += st["scale"] * ((x @ a.t()) @ b.t())
        if st["bias"] is not None:
            y += st["bias"].float()
        return {"y": y.to(st["x"].dtype)}
    dy, r = st["dy"].float(), a.shape[0]
    half = st["z"].shape[1] // 2
    z = st["z"][:, :r].float() + st["z"][:, half:half + r].float()
    grad = st["scale"] * (dy @ b)
    dtype = st["dy"].dtype
    out = {"dx": None, "da": (grad.t() @ _decode(st["x8"])).to(dtype), "db": (dy.t() @ z).to(dtype)}
    if st["dx"]:
        out["dx"] = (dy @ _decode(st["w"]) + grad @ a).to(dtype)
    return out


def run(st):
    return _run_own(st) if own else _run_plain(st)


def work(case):
    """The pass's bytes, each input read once and each output written once, and its products."""
    m, k, op = case["m"], case["k"], case["op"]
    kp = (k + 31) // 32 * 32
    if op in ("quantize", "checkpoint"):
        per = {"mxfp4": 0.5 + 1 / 32, "nvfp4": 0.5 + 1 / 16, "mxfp8": 1 + 1 / 32}[case.get("fmt", "mxfp8")]
        # x in, codes and scales out and in again, values out
        return {"bytes": 4 * m * k + 2 * per * m * kp, "flops": 0}
    n, r = case["n"], case["r"]
    per = {"mxfp4": 0.5 + 1 / 32, "nvfp4": 0.5 + 1 / 16}[case["fmt"]]
    wb, ab = per * n * kp, 2 * r * (n + k)
    if op == "linear":
        return {"bytes": 2 * m * (k + n) + wb + ab + (2 * n if case["bias"] else 0),
                "flops": 2 * m * n * k + 2 * m * r * (n + k)}
    r16 = (r + 15) // 16 * 16
    by = 2 * m * n + (1 + 1 / 32) * m * kp + 4 * m * r16 + 2 * ab
    fl = 4 * m * r * n + 2 * m * r * k
    if case["dx"]:
        by += wb + 2 * m * k
        fl += 2 * m * n * k + 2 * m * r * k
    return {"bytes": by, "flops": fl}


# --------------------------------------------------- the same from the definition, in 64 bits
_E2M1 = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]


def _grid_e4m3():
    return [i / 512.0 for i in range(8)] + [(1 + j / 8.0) * 2.0 ** e for e in range(-6, 9) for j in range(8)][:-1]


def _nearest64(y, grid):
    """The nearest value of the grid, ties to the one of even index, the largest beyond it."""
    t = torch.tensor(grid, dtype=torch.float64, device=y.device)
    mids = (t[1:] + t[:-1]) / 2
    a = y.abs()
    lo, hi = torch.searchsorted(mids, a, right=False), torch.searchsorted(mids, a, right=True)
    i = torch.where(lo == hi, lo, torch.where(lo % 2 == 0, lo, hi))
    return torch.copysign(t[i], y)


def _values64(x, fmt, g):
    m, k = x.shape
    size = BLOCK[fmt]
    out = torch.empty(m, k, dtype=torch.float64, device=x.device)
    for r0 in range(0, m, 4096):  # in parts: the search over the grid holds several copies
        v = torch.nn.functional.pad(x[r0:r0 + 4096].double(), (0, -k % size)).unflatten(1, (-1, size))
        top = v.abs().amax(2, keepdim=True)
        if fmt == "nvfp4":
            unit = _nearest64(top / (6 * g), _grid_e4m3()) * g
            q = torch.where(unit > 0, _nearest64(v / torch.where(unit > 0, unit, 1.0), _E2M1), 0.0)
        else:
            emax = 2 if fmt == "mxfp4" else 8
            unit = torch.ldexp(torch.ones_like(top), torch.clamp(torch.frexp(top).exponent - 1 - emax, min=-127))
            q = _nearest64(v / unit, _E2M1 if fmt == "mxfp4" else _grid_e4m3())
        out[r0:r0 + 4096] = (q * unit).flatten(1)[:, :k]
    return out


def _held64(t):
    m, k = t["shape"]
    e4 = torch.tensor(_grid_e4m3() + [math.nan], dtype=torch.float64, device=DEV)
    e4 = torch.cat([e4, -e4])
    e2 = torch.tensor(_E2M1, dtype=torch.float64, device=DEV)
    e2 = torch.cat([e2, -e2])
    c = t["codes"].long()
    q = e4[c] if t["fmt"] == "mxfp8" else torch.stack([e2[c % 16], e2[c // 16]], 2).flatten(1)
    size = BLOCK[t["fmt"]]
    nb = q.shape[1] // size
    row = torch.arange(m, device=DEV)[:, None]
    blk = torch.arange(nb, device=DEV)[None, :]
    chunk = (row // 128) * ((nb + 3) // 4) + blk // 4
    s = t["scales"][chunk * 512 + (row % 32) * 16 + (row % 128) // 32 * 4 + blk % 4].long()
    s = e4[s] if t["fmt"] == "nvfp4" else torch.pow(2.0, s.double() - 127)
    return (q.unflatten(1, (nb, size)) * s[:, :, None]).flatten(1)[:, :k] * t["global_scale"]


def exact(case, seed):
    st = prepare(case, seed)
    if st["op"] in ("quantize", "checkpoint"):
        return {"values": _values64(st["x"], st["fmt"], st["global_scale"])}
    a, b, s = st["a"].double(), st["b"].double(), st["scale"]
    if st["op"] == "linear":
        y = _values64(st["x"], st["w"]["fmt"], st["x_global"]) @ _held64(st["w"]).T
        y.addmm_(st["x"].double() @ (s * a).T, b.T)
        return {"y": y if st["bias"] is None else y.add_(st["bias"].double())}
    dy, r = st["dy"].double(), a.shape[0]
    zz = st["z"].double().unflatten(1, (2, -1)).sum(1)[:, :r]
    u = dy @ (s * b)
    return {"dx": torch.addmm(u @ a, dy, _held64(st["w"])) if st["dx"] else None,
            "da": u.T @ _held64(st["x8"]), "db": dy.T @ zz}
