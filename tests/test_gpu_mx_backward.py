"""Gradients of the 4-bit LoRA linear from the 8-bit checkpoint of its input.

Against the float64 formulas on the stored values, against differences of the
float64 forward pass, and through autograd.
"""

import numpy as np
import pytest
import torch
from torch import nn

from oracle import mx_oracle as mo
from probe_b200 import _lib, mx
from tests.helpers import dtype_tag, np64, randn

pytestmark = pytest.mark.gpu
DEV = "cuda"
GW = {"mxfp4": 1.0, "nvfp4": float(np.float32(0.31 / 2688))}


def case(m, n, k, r, dtype, fmt="mxfp4", seed=0):
    r16 = (r + 15) // 16 * 16
    dy = randn((m, n), 1.0, dtype, seed)
    x8 = mx.mx_quantize(randn((m, k), 2.0, dtype, seed + 1), "mxfp8")
    zf = randn((m, r), 1.5, torch.float32, seed + 2)
    z = torch.zeros(m, 2 * r16, dtype=dtype, device=DEV)
    z[:, :r] = zf.to(dtype)
    z[:, r16:r16 + r] = zf - z[:, :r].float()
    a, b = randn((r, k), k ** -0.5, dtype, seed + 3), randn((n, r), max(r, 1) ** -0.5, dtype, seed + 4)
    return dy, x8, z, a, b, mx.mx_quantize(randn((n, k), k ** -0.5, dtype, seed + 5), fmt, GW[fmt])


def values(q):
    """Float64 values of a stored tensor, decoded by the oracle's grids and layout."""
    m, k = q.shape
    c = q.codes.cpu().numpy()
    if q.fmt == "mxfp8":
        grid, sign, mag = np.append(mo.E4M3, np.nan), c >> 7, c & 0x7F
    else:
        c = np.stack([c & 15, c >> 4], axis=2).reshape(m, -1)
        grid, sign, mag = mo.E2M1, c >> 3, c & 7
    v = np.where(sign == 1, -grid[mag], grid[mag])
    size = mo.BLOCK[q.fmt]
    nb = v.shape[1] // size
    s, row, blk = q.scales.cpu().numpy(), np.arange(m)[:, None], np.arange(nb)[None]
    byte = s[(row // 128 * (-(-nb // 4)) + blk // 4) * 512 + row % 32 * 16 + row % 128 // 32 * 4 + blk % 4].astype(int)
    sc = np.append(mo.E4M3, np.nan)[byte] if q.fmt == "nvfp4" else np.where(byte == 255, np.nan, 2.0 ** (byte - 127.0))
    return (v.reshape(m, nb, size) * sc[:, :, None]).reshape(m, -1)[:, :k] * q.global_scale


def formulas(dy, x8, z, a, b, w, scale, z_scale, dtype):
    """(reference, elementwise bound) of da, db and dx."""
    d, xv, av, bv = np64(dy), values(x8), np64(a), np64(b)
    m, n = d.shape
    r = av.shape[0]
    r16 = z.shape[1] // 2
    tag = dtype_tag(dtype)
    # the halves of z and of g that the products read: the pair up to rank 64 (error
    # 2^-16 of a value in bf16, 2^-22 in fp16), one rounding above
    eps = (2.0 ** -8 if tag == "bf16" else 2.0 ** -11)
    pair = eps * eps if r16 <= 64 else eps
    zv = z_scale * (np64(z[:, :r]) + np64(z[:, r16:r16 + r]))
    g = scale * d @ bv
    gacc = (n / 16 + 8) * 2.0 ** -23 * abs(scale) * (np.abs(d) @ np.abs(bv))  # g's own float32 sum
    da, dam = g.T @ xv, np.abs(g).T @ np.abs(xv)
    db, dbm = d.T @ zv, np.abs(d).T @ np.abs(zv)
    out = {
        "da": (da, mo.product_bound(da, dam, m, tag, pair * dam + gacc.T @ np.abs(xv))),
        "db": (db, mo.product_bound(db, dbm, m, tag, pair * dbm)),
    }
    if w is not None:
        wv = values(w)
        dx = d @ wv + g @ av
        lora = np.abs(g) @ np.abs(av)
        out["dx"] = (dx, mo.product_bound(dx, np.abs(d) @ np.abs(wv) + lora, n + 2 * r16, tag,
                                          eps * eps * lora + gacc @ np.abs(av)))
    return out


def check(got, want):
    for name, t in zip(("dx", "da", "db"), got):
        if name not in want:
            assert t is None
            continue
        ref, bound = want[name]
        err = np.abs(np64(t) - ref)
        assert t.shape == ref.shape and np.isfinite(np64(t)).all(), name
        assert (err <= bound).all(), f"{name}: worst {np.max(err / bound):.2f} of the bound"


SIZES = [(1, 64, 32, 4), (1, 8, 256, 64), (2, 257, 96, 1), (63, 128, 130, 16), (64, 256, 256, 48), (65, 520, 288, 65),
         (130, 1001, 544, 20), (300, 96, 1000, 224), (513, 264, 520, 256), (1030, 2304, 320, 8), (2600, 136, 264, 130),
         (4100, 264, 288, 200), (4097, 130, 160, 16)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("fmt", ["mxfp4", "nvfp4"])
@pytest.mark.parametrize("m,n,k,r", SIZES)
def test_against_formulas(m, n, k, r, fmt, dtype):
    dy, x8, z, a, b, w = case(m, n, k, r, dtype, fmt)
    got = mx.mx_lora_backward(dy, x8, z, a, b, 1.7, weight=w, z_scale=1.25)
    check(got, formulas(dy, x8, z, a, b, w, 1.7, 1.25, dtype))
    assert _lib.device_error(0) == 0


@pytest.mark.parametrize("m,n,k,r", [(100, 200, 160, 12), (700, 512, 512, 224)])
def test_without_dx(m, n, k, r):
    dy, x8, z, a, b, w = case(m, n, k, r, torch.bfloat16)
    with_dx = mx.mx_lora_backward(dy, x8, z, a, b, 0.5, weight=w)
    got = mx.mx_lora_backward(dy, x8, z, a, b, 0.5)
    check(got, formulas(dy, x8, z, a, b, None, 0.5, 1.0, torch.bfloat16))
    assert torch.equal(got[1], with_dx[1]) and torch.equal(got[2], with_dx[2])


def test_against_differences():
    """The formulas are the derivatives of the forward pass: central differences of
    sum(dy * (X W^T + s (X A^T) B^T)) in float64, at a few entries of A, B and X."""
    m, n, k, r, s = 6, 40, 64, 4, 1.5
    dy, x8, z, a, b, w = case(m, n, k, r, torch.float16)
    xv, wv, av, bv, d = values(x8), values(w), np64(a), np64(b), np64(dy)
    zv = s * xv @ av.T
    r16 = z.shape[1] // 2
    zt = torch.from_numpy(zv).float().to(DEV)
    z.zero_()
    z[:, :r] = zt.half()
    z[:, r16:r16 + r] = zt - z[:, :r].float()

    def loss(xv, av, bv):
        return float((d * (xv @ wv.T + s * (xv @ av.T) @ bv.T)).sum())

    dx, da, db = mx.mx_lora_backward(dy, x8, z, a, b, s, weight=w)
    want = formulas(dy, x8, z, a, b, w, s, 1.0, torch.float16)
    h = 2.0 ** -10  # the loss is linear in each of them: differences are exact up to rounding
    rng = np.random.RandomState(0)
    for name, got, at in (("dx", dx, 0), ("da", da, 1), ("db", db, 2)):
        for _ in range(12):
            args = [xv.copy(), av.copy(), bv.copy()]
            i = tuple(rng.randint(0, v) for v in args[at].shape)
            args[at][i] += h
            up = loss(*args)
            args[at][i] -= 2 * h
            diff = (up - loss(*args)) / (2 * h)
            bound = want[name][1][i] + 1e-8 * abs(up)
            assert abs(float(got[i]) - diff) <= bound, (name, i)


def test_layouts_and_streams():
    m, n, k, r = 200, 320, 256, 24
    dy, x8, z, a, b, w = case(m, n, k, r, torch.bfloat16)
    base = mx.mx_lora_backward(dy, x8, z, a, b, 2.0, weight=w)
    wide = torch.zeros(m, n + 9, dtype=dy.dtype, device=DEV)
    wide[:, 5:5 + n] = dy
    bt = torch.zeros(n, r + 3, dtype=dy.dtype, device=DEV)
    bt[:, 2:2 + r] = b
    want = formulas(dy, x8, z, a, b, w, 2.0, 1.0, torch.bfloat16)
    check(mx.mx_lora_backward(wide[:, 5:5 + n], x8, z, a.t().contiguous().t(), bt[:, 2:2 + r], 2.0, weight=w), want)
    s = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(s):
        other = mx.mx_lora_backward(dy.view(2, m // 2, n), x8, z, a, b, 2.0, weight=w)
    s.synchronize()
    assert other[0].shape == (2, m // 2, k)
    for p, q in zip(base, other):
        assert torch.equal(p.reshape(-1), q.reshape(-1))
    for _ in range(3):
        for p, q in zip(base, mx.mx_lora_backward(dy, x8, z, a, b, 2.0, weight=w)):
            assert torch.equal(p, q)


def test_large_and_small_checkpoint_scales():
    """Scales on both sides of the one-multiply decode (2^7), zeros and subnormal codes."""
    m, n, k, r = 96, 64, 128, 16
    dy, _, z, a, b, _ = case(m, n, k, r, torch.bfloat16)
    x = randn((m, k), 1.0, torch.bfloat16, 9)
    x[:, :32] *= 2.0 ** 18
    x[:, 32:64] *= 2.0 ** -30
    x[:, 64:96] *= torch.exp2(torch.randint(-14, 1, (m, 32), device=DEV).float()).to(x.dtype)
    x[5] = 0
    x8 = mx.mx_quantize(x, "mxfp8")
    check(mx.mx_lora_backward(dy, x8, z, a, b, 1.0), formulas(dy, x8, z, a, b, None, 1.0, 1.0, torch.bfloat16))


def test_a_nan_block_of_the_checkpoint_reaches_its_columns_only():
    m, n, k, r = 80, 64, 160, 8
    dy, _, z, a, b, w = case(m, n, k, r, torch.bfloat16)
    x = randn((m, k), 1.0, torch.bfloat16, 7)
    clean = mx.mx_lora_backward(dy, mx.mx_quantize(x, "mxfp8"), z, a, b, 1.0)
    x[3, 40] = float("inf")
    _, da, db = mx.mx_lora_backward(dy, mx.mx_quantize(x, "mxfp8"), z, a, b, 1.0)
    assert da[:, 32:64].isnan().all() and torch.equal(db, clean[2])
    assert torch.equal(da[:, :32], clean[1][:, :32]) and torch.equal(da[:, 64:], clean[1][:, 64:])


def test_empty_batch_has_zero_gradients():
    dy, x8, z, a, b, w = case(4, 64, 96, 8, torch.bfloat16)
    none = mx.mx_quantize(torch.zeros(0, 96, dtype=torch.bfloat16, device=DEV), "mxfp8")
    dx, da, db = mx.mx_lora_backward(dy[:0], none, z[:0], a, b, 1.0, weight=w)
    assert dx.shape == (0, 96) and not da.any() and not db.any()


def test_refusals():
    dy, x8, z, a, b, w = case(8, 64, 96, 8, torch.bfloat16)
    with pytest.raises(ValueError, match="mxfp8"):
        mx.mx_lora_backward(dy, w, z, a, b)
    with pytest.raises(ValueError, match="pair"):
        mx.mx_lora_backward(dy, x8, z[:, :16].contiguous(), a, b)
    with pytest.raises(TypeError):
        mx.mx_lora_backward(dy.half(), x8, z, a, b)
    with pytest.raises(TypeError):
        mx.mx_lora_backward(dy.float(), x8, z, a, b)
    with pytest.raises(ValueError):
        mx.mx_lora_backward(dy, x8, z, a, b[:32])
    with pytest.raises(ValueError, match="4-bit"):
        mx.mx_lora_backward(dy, x8, z, a, b, weight=x8)
    with pytest.raises(RuntimeError, match="CUDA"):
        mx.mx_lora_backward(dy.cpu(), x8, z, a, b)


# -------------------------------------------------------------------------- module
def module(n=192, k=256, r=12, fmt="mxfp4", dtype=torch.bfloat16, bias=True, seed=0):
    base = nn.Linear(k, n, bias=bias, device=DEV, dtype=dtype)
    with torch.no_grad():
        base.weight.copy_(randn((n, k), k ** -0.5, dtype, seed))
    a, b = randn((r, k), k ** -0.5, dtype, seed + 1), randn((n, r), r ** -0.5, dtype, seed + 2)
    return mx.MXLoRALinear(base, a, b, 1.5, fmt)


@pytest.mark.parametrize("fmt", ["mxfp4", "nvfp4"])
@pytest.mark.parametrize("m", [5, 300])
def test_module_gradients(m, fmt):
    mod = module(fmt=fmt)
    x = randn((1, m, 256), 1.0, torch.bfloat16, 5).requires_grad_()
    dy = randn((1, m, 192), 1.0, torch.bfloat16, 6)
    y = mod(x)
    with torch.no_grad():
        assert torch.equal(y, mod(x))
    y.backward(dy)
    flat = x.detach().view(m, 256)
    _, x8, z, zs = mx.mx_lora_forward(flat, mod.weight, mod.bias, mod.lora_a, mod.lora_b, 1.5, mod.x_global_scale)
    want = formulas(dy[0], x8, z, mod.lora_a, mod.lora_b, mod.weight, 1.5, zs, torch.bfloat16)
    check((x.grad[0], mod.lora_a.grad, mod.lora_b.grad), want)
    r = mod.rank
    r16 = z.shape[1] // 2
    zt = zs * (np64(z[:, :r]) + np64(z[:, r16:r16 + r]))
    exact = 1.5 * np64(flat) @ np64(mod.lora_a).T
    mass = 1.5 * np.abs(np64(flat)) @ np.abs(np64(mod.lora_a)).T
    assert (np.abs(zt - exact) <= 2.0 ** -16 * np.abs(exact) + 24 * 2.0 ** -23 * mass).all()


def test_module_trains_and_serves():
    """A few steps of gradient descent on the adapter alone, then greedy use without gradients."""
    mod = module(seed=3)
    codes = mod.w_codes.clone()
    x = randn((256, 256), 1.0, torch.bfloat16, 8)
    target = randn((256, 192), 1.0, torch.bfloat16, 9)
    opt = torch.optim.SGD([p for p in mod.parameters()], lr=2e-3)
    losses = []
    for _ in range(12):
        opt.zero_grad()
        loss = (mod(x) - target).float().square().mean(1).sum()
        loss.backward()
        opt.step()
        losses.append(float(loss))
    assert losses[-1] < 0.97 * losses[0] and torch.equal(codes, mod.w_codes)
    with torch.no_grad():
        assert mod(x[:1]).shape == (1, 192)


def test_module_leaves_out_what_is_not_asked_for():
    mod = module()
    x = randn((40, 256), 1.0, torch.bfloat16, 5)
    mod(x).sum().backward()
    assert mod.lora_a.grad is not None and mod.lora_b.grad is not None
    mod.lora_a.requires_grad_(False)
    mod.lora_a.grad = None
    mod(x).sum().backward()
    assert mod.lora_a.grad is None
    saved = []
    with torch.autograd.graph.saved_tensors_hooks(lambda t: saved.append(t) or t, lambda t: t):
        mod(x)
    # codes, scales, z and the two factors: nothing 16-bit of x's size
    assert not any(t.shape == x.shape and t.dtype == x.dtype for t in saved)


def test_module_refusals():
    base = nn.Linear(64, 32, device=DEV, dtype=torch.bfloat16)
    a, b = torch.zeros(4, 64), torch.zeros(32, 4)
    with pytest.raises(ValueError, match="fmt"):
        mx.MXLoRALinear(base, a, b, fmt="mxfp8")
    with pytest.raises(ValueError, match="do not match"):
        mx.MXLoRALinear(base, a[:, :32], b)


def test_from_a_fresh_host_thread():
    """A thread whose first CUDA work is the call itself (its tensors come from the allocator's cache)."""
    import threading

    dy, x8, z, a, b, w = case(130, 192, 256, 12, torch.bfloat16)
    want = mx.mx_lora_backward(dy, x8, z, a, b, 1.0, weight=w)
    torch.cuda.synchronize()
    got = []
    t = threading.Thread(target=lambda: got.append(mx.mx_lora_backward(dy, x8, z, a, b, 1.0, weight=w)))
    t.start()
    t.join()
    assert len(got) == 1 and all(torch.equal(p, q) for p, q in zip(got[0], want))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("fmt", ["mxfp4", "nvfp4"])
@pytest.mark.parametrize("m,n,k,r", [(300, 72, 9608, 20), (4097, 136, 1288, 224), (260, 65, 9601, 5)])
def test_many_output_tiles(m, n, k, r, fmt, dtype):
    """dx of more tiles than the kernel that decodes W on the way takes."""
    dy, x8, z, a, b, w = case(m, n, k, r, dtype, fmt, seed=3)
    got = mx.mx_lora_backward(dy, x8, z, a, b, 0.7, weight=w, z_scale=1.25)
    check(got, formulas(dy, x8, z, a, b, w, 0.7, 1.25, dtype))


@pytest.mark.parametrize("m", [15, 16, 17, 32, 33, 64, 65, 128, 129, 256, 257, 600])
@pytest.mark.parametrize("fmt,n,k,r", [("mxfp4", 63, 96, 16), ("nvfp4", 1090, 200, 72)])
def test_row_tiles(m, fmt, n, k, r):
    dy, x8, z, a, b, w = case(m, n, k, r, torch.bfloat16, fmt, seed=7)
    got = mx.mx_lora_backward(dy, x8, z, a, b, 1.0, weight=w)
    check(got, formulas(dy, x8, z, a, b, w, 1.0, 1.0, torch.bfloat16))


@pytest.mark.parametrize("m", [20, 300])
@pytest.mark.parametrize("fmt", ["mxfp4", "nvfp4"])
def test_weight_scales_far_from_one(m, fmt):
    """Blocks of W whose scale is huge, tiny or zero, side by side; tensor scales likewise."""
    n, k, r = 136, 256, 16
    dy, x8, z, a, b, _ = case(m, n, k, r, torch.bfloat16, fmt, seed=11)
    wf = randn((n, k), k ** -0.5, torch.bfloat16, 21)
    if fmt == "mxfp4":
        wf[:, :32] *= 2.0 ** 90
        wf[:, 32:64] *= 2.0 ** -100
        wf[:, 64:96] = 0
        weights = [mx.mx_quantize(wf, fmt)]
    else:
        weights = [mx.mx_quantize(wf * 2.0 ** e, fmt, GW[fmt] * 2.0 ** e) for e in (50, -40)]
    for w in weights:
        got = mx.mx_lora_backward(dy, x8, z, a, b, 1.0, weight=w)
        check(got, formulas(dy, x8, z, a, b, w, 1.0, 1.0, torch.bfloat16))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("fmt", ["mxfp4", "nvfp4"])
def test_a_nan_block_of_the_weight_reaches_its_columns_only(fmt, dtype):
    m, n, k, r = 70, 200, 256, 8
    dy, x8, z, a, b, w = case(m, n, k, r, dtype, fmt, seed=5)
    wf = randn((n, k), k ** -0.5, dtype, 10)
    wf[77, 101] = float("inf")
    bad = mx.mx_quantize(wf, fmt, GW[fmt])
    dx, _, _ = mx.mx_lora_backward(dy, x8, z, a, b, 1.0, weight=bad)
    size = mo.BLOCK[fmt]
    hit = torch.zeros(k, dtype=torch.bool, device=DEV)
    hit[101 // size * size:101 // size * size + size] = True
    assert torch.isnan(dx[:, hit]).all() and torch.isfinite(dx[:, ~hit]).all()


@pytest.mark.parametrize("m", [20, 300])
@pytest.mark.parametrize("fmt", ["mxfp4", "nvfp4"])
@pytest.mark.parametrize("e", [-12, 9])
def test_weight_values_at_the_ends_of_fp16(m, fmt, e):
    """Scales below fp16's normal numbers (values that it still holds exactly) and large ones."""
    n, k, r = 136, 256, 16
    dy, x8, z, a, b, _ = case(m, n, k, r, torch.float16, fmt, seed=13)
    dy, a = dy * 2.0 ** -e, torch.zeros_like(a)
    wf = randn((n, k), k ** -0.5, torch.float16, 23) * 2.0 ** e
    w = mx.mx_quantize(wf, fmt, 1.0 if fmt == "mxfp4" else 2.0 ** (e - 11))
    got = mx.mx_lora_backward(dy, x8, z, a, b, 2.0 ** -6, weight=w)
    want = formulas(dy, x8, z, a, b, w, 2.0 ** -6, 1.0, torch.float16)
    check((got[0],), {"dx": want["dx"]})
