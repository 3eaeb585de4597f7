"""Layer norm and counter-based dropout from their definitions in 64 bits, with bounds on what 32-bit arithmetic
and the one rounding of the result may be off by."""
import numpy as np
import torch

U = 2.0 ** -24                                     # half a step of float32


def philox(ctr, key, rounds=7):
    """Philox4x32 on arrays of 32-bit words held in uint64"""
    low = np.uint64(0xFFFFFFFF)
    s = np.uint64(32)
    c = [np.asarray(v, np.uint64) for v in ctr]
    k0, k1 = key
    for i in range(rounds):
        a, b = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        x0 = np.uint64((k0 + i * 0x9E3779B9) & 0xFFFFFFFF)
        x1 = np.uint64((k1 + i * 0xBB67AE85) & 0xFFFFFFFF)
        c = [(b >> s) ^ c[1] ^ x0, b & low, (a >> s) ^ c[3] ^ x1, a & low]
    return c


def keep_mask(rows, dim, p, seed, step=0, row_offset=0):
    """[rows, dim] truth values"""
    if p == 0:
        return np.ones((rows, dim), bool)
    e = np.arange(row_offset * dim, (row_offset + rows) * dim, dtype=np.uint64)
    g, low = e >> np.uint64(2), np.uint64(0xFFFFFFFF)
    one = np.ones_like(g)
    words = philox([g & low, g >> np.uint64(32), one * np.uint64(step & 0xFFFFFFFF), one * np.uint64(step >> 32)],
                   (seed & 0xFFFFFFFF, seed >> 32))
    pick = (e & np.uint64(3)).astype(np.int64)
    word = np.stack(words, 1)[np.arange(e.size), pick]
    return (word >= np.uint64(round(p * 2 ** 32))).reshape(rows, dim)


def tiny(dtype):
    """half a step of the type's smallest values: float16 holds what is below 2^-14 in steps of 2^-24"""
    return 2.0 ** -25 if dtype == torch.float16 else 1e-37


def _f64(t):
    return None if t is None else t.detach().double().cpu().numpy()


def z_of(x, w, b, eps):
    x = _f64(x)
    h = (x - x.mean(-1, keepdims=True)) / np.sqrt(x.var(-1, keepdims=True) + eps)
    return h * (_f64(w) if w is not None else 1.0) + (_f64(b) if b is not None else 0.0)


def norm_reference(x, w, b, eps=1e-5, relu=False, p=0.0, seed=0, step=0, row_offset=0, dy=None):
    """-> {name: (value, bound)} of y and, with dy, of dx, dw, db; [rows, dim] inputs.

    The bounds.  Every sum over a row of D adds at most D/32 + 16 terms one after the other (gamma below).  The mean is a first
    value m plus sum(x - m) / D: the addition and each x - m are rounded (values of the size of x), and the sum is off by at most
    gamma times mean |x - m| <= gamma / rstd, which is gamma in units of h = (x - mean) rstd; rstd is off by gamma of itself, so
    h by gamma |h| more.  Products and differences of single elements add a few roundings each.  A sum over the rows adds at most
    1100 + rows/1024 terms one after the other."""
    half = torch.finfo(x.dtype).eps / 2
    vtype = w.dtype if w is not None else torch.float32
    vhalf = torch.finfo(vtype).eps / 2
    X, W, B = _f64(x), _f64(w), _f64(b)
    n, d = X.shape
    W1, B0 = (W if W is not None else np.ones(d)), (B if B is not None else np.zeros(d))
    mean = X.mean(1, keepdims=True)
    rstd = 1.0 / np.sqrt(((X - mean) ** 2).mean(1, keepdims=True) + eps)
    h = (X - mean) * rstd
    z = h * W1 + B0
    keep = keep_mask(n, d, p, seed, step, row_offset)
    s = 1.0 / (1.0 - p) if p < 1 else 0.0
    a = np.maximum(z, 0.0) if relu else z
    y = np.where(keep, a * s, 0.0)
    gamma = (d / 32 + 16) * U
    eh = 4 * U * (np.abs(X) + np.abs(mean)) * rstd + gamma * (1 + np.abs(h))
    out = {"y": (y, half * np.abs(y) + s * (np.abs(W1) * eh + 4 * U * (np.abs(h * W1) + np.abs(B0))) + tiny(x.dtype))}
    if dy is None:
        return out
    dz = np.where(keep, _f64(dy) * s, 0.0)
    if relu:
        dz = np.where(z > 0, dz, 0.0)
    g = dz * W1
    c1, c2 = g.mean(1, keepdims=True), (g * h).mean(1, keepdims=True)
    dx = rstd * (g - c1 - h * c2)
    size = np.abs(g) + np.abs(g).mean(1, keepdims=True) + np.abs(h) * np.abs(g * h).mean(1, keepdims=True)
    e_dx = rstd * ((gamma + 8 * U) * size + np.abs(h) * (np.abs(g) * eh).mean(1, keepdims=True) + eh * np.abs(g * h).mean(1, keepdims=True))
    out["dx"] = (dx, half * np.abs(dx) + e_dx + tiny(x.dtype))
    depth = min(n, 1100 + n / 1024) + 4
    dw, db = (dz * h).sum(0), dz.sum(0)
    out["dw"] = (dw, vhalf * np.abs(dw) + (np.abs(dz) * eh).sum(0) + depth * U * np.abs(dz * h).sum(0) + tiny(vtype))
    out["db"] = (db, vhalf * np.abs(db) + depth * U * np.abs(dz).sum(0) + tiny(vtype))
    return out


def dropout_reference(x, bias=None, relu=False, p=0.0, seed=0, step=0, row_offset=0, dy=None):
    half = torch.finfo(x.dtype).eps / 2
    X, B = _f64(x), _f64(bias)
    n, d = X.shape
    z = X if B is None else X + B
    keep = keep_mask(n, d, p, seed, step, row_offset)
    s = 1.0 / (1.0 - p) if p < 1 else 0.0
    a = np.maximum(z, 0.0) if relu else z
    y = np.where(keep, a * s, 0.0)
    # the sum, the scale and the product are rounded to 32 bits, the result to its type
    out = {"y": (y, (half + 3 * U) * np.abs(y) + tiny(x.dtype))}
    if dy is None:
        return out
    dz = np.where(keep, _f64(dy) * s, 0.0)
    if relu:
        dz = np.where(z > 0, dz, 0.0)
    out["dx"] = (dz, (half + 3 * U) * np.abs(dz) + tiny(x.dtype))
    if B is not None:
        vhalf = torch.finfo(bias.dtype).eps / 2
        depth = min(n, 1100 + n / 1024) + 4
        db = dz.sum(0)
        out["db"] = (db, vhalf * np.abs(db) + depth * U * np.abs(dz).sum(0) + tiny(bias.dtype))
    return out


def assert_within(got, want, what=""):
    value, bound = want
    g = got.detach().double().cpu().numpy().reshape(value.shape)
    err = np.abs(g - value)
    bad = ~(err <= bound)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.size} off, worst {np.nanmax(err / bound):.3g} of the bound, nan {np.isnan(g).sum()}"
