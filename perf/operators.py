"""Measured cases of the operators between two graph layers: layer norm, dropout from a counter-based
generator, and the two joined with the ReLU between them.

A case's `op` is "norm" (layer norm), "dropout" (optionally with the bias add and the ReLU that stand before it
in a GCN stack) or "hidden" (dropout of the ReLU of a layer norm).  `pass` is "forward" (serving) or "train" (the
outputs and the gradients of all inputs).  `pad` gives the rows of the inputs the stride that keeps them 16-byte
aligned, as the framework's own padded buffers have.

The generator is Philox4x32 with seven rounds (Salmon et al., "Parallel random numbers: as easy as 1, 2, 3",
SC 2011): element e of the row-major matrix takes word e % 4 of counter (e / 4, step) under the key `seed` and is
dropped where the word is below p * 2^32.
"""
import math

import torch

own = False

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
EPS = 1e-5
MOST_ELEMENTS = 2449029 * 256          # the largest matrix of the repository's own configurations


def _case(name, op, direction, rows, dim, dtype="f32", p=0.0, bias=False, relu=False, pad=False):
    return {"name": name, "op": op, "pass": direction, "rows": rows, "dim": dim, "dtype": dtype, "p": p, "bias": bias,
            "relu": relu, "pad": pad}


def listed():
    return [
        # one node served: the latency of a call
        _case("norm-forward-1x128", "norm", "forward", 1, 128),
        # the citation graph (2,708 nodes, 16 hidden features): a training step bound by launches
        _case("norm-train-2708x16", "norm", "train", 2708, 16),
        # the post graph at its raw feature width; rows of 2,408 bytes, not 16-byte aligned
        _case("norm-train-232965x602", "norm", "train", 232965, 602),
        # the product graph at the width of its hidden layers: the largest matrix
        _case("norm-train-2449029x256", "norm", "train", 2449029, 256),
        # the product graph at its number of classes, served in 16 bits: odd rows
        _case("norm-forward-2449029x47-bf16", "norm", "forward", 2449029, 47, "bf16"),
        # wide rows of a 16-bit MLP
        _case("norm-train-16384x4096-bf16", "norm", "train", 16384, 4096, "bf16"),
        # dropout between the layers of the citation graph's stack
        _case("dropout-train-2708x16", "dropout", "train", 2708, 16, p=0.5),
        # the community graph (2^20 nodes, 64 features)
        _case("dropout-train-1048576x64", "dropout", "train", 1048576, 64, p=0.3),
        # what stands between two layers of a GCN stack on the post graph: bias, ReLU, dropout
        _case("dropout-train-bias-relu-232965x256", "dropout", "train", 232965, 256, p=0.5, bias=True, relu=True),
        # the product graph's raw features in 16 bits
        _case("dropout-train-2449029x100-f16", "dropout", "train", 2449029, 100, "f16", p=0.1),
        # a normed hidden layer on the paper graph
        _case("hidden-train-169343x128", "hidden", "train", 169343, 128, p=0.5, relu=True),
        # a normed hidden layer of odd width on the product graph
        _case("hidden-train-2449029x47", "hidden", "train", 2449029, 47, p=0.2, relu=True),
    ]


def _log_int(rng, low, high):
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["norm", "dropout", "hidden"])
    dim = _log_int(rng, 8, 4096)
    if rng.random() < 0.4:
        dim = max(8, dim // 8 * 8)
    rows = _log_int(rng, 1, min(2449029, (MOST_ELEMENTS if op == "norm" else MOST_ELEMENTS // 4) // dim))
    case = _case("", op, rng.choice(["forward", "train", "train"]), rows, dim, rng.choice(["f32", "f32", "bf16", "f16"]),
                 0.0 if op == "norm" else rng.choice([0.1, 0.2, 0.5, 0.6]), op == "dropout" and rng.random() < 0.5,
                 op == "hidden" or (op == "dropout" and rng.random() < 0.5), rng.random() < 0.3)
    if op == "hidden" and case["pass"] == "forward" and rng.random() < 0.5:
        case["p"] = 0.0                                      # serving: no dropout
    del case["name"]
    return case


def _rows(values, case):
    """`values` in the case's type, with the case's row stride"""
    values = values.to(TYPES[case["dtype"]])
    if not case["pad"]:
        return values
    per = 16 // values.element_size()
    buf = torch.empty((case["rows"], -(-case["dim"] // per) * per), dtype=values.dtype, device=values.device)
    view = buf[:, :case["dim"]]
    view.copy_(values)
    return view


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev)
    gen.manual_seed(seed)
    n, d = case["rows"], case["dim"]
    randn = lambda *s: torch.randn(*s, generator=gen, device=dev)  # noqa: E731
    # aggregated features: every column its own offset, every row its own scale
    x = randn(n, d)
    x.mul_(0.5 + torch.rand(n, 1, generator=gen, device=dev) * 2).add_(0.3 * randn(1, d))
    s = {"case": case, "x": _rows(x, case), "w": None, "b": None, "dy": None,
         "seed": int(torch.randint(0, 2 ** 62, (1,), generator=gen, device=dev)), "step": int(seed) % 1000}
    del x
    if case["op"] != "dropout":
        s["w"], s["b"] = 1.0 + 0.2 * randn(d), 0.2 * randn(d)
    elif case["bias"]:
        s["b"] = 0.2 * randn(d)
    if case["pass"] == "train":
        dy = randn(n, d)
        if case["op"] == "hidden":
            # next to the ReLU's border a rounding decides which one-sided gradient holds: no gradient comes in there
            step = max(1, (1 << 26) // d)
            for i in range(0, n, step):
                v = s["x"][i:i + step].double()
                v = v - v.mean(1, keepdim=True)
                v = v / (v.square().mean(1, keepdim=True) + EPS).sqrt() * s["w"].double() + s["b"].double()
                dy[i:i + step].masked_fill_(v.abs() < 2e-5, 0.0)
                del v
        s["dy"] = _rows(dy, case)
        for k in ("x", "w", "b"):
            if s[k] is not None:
                s[k].requires_grad_(True)
    return s


# ---- plain form ---------------------------------------------------------------------------------
def _round(c0, c1, c2, c3, k0, k1):
    """one round of Philox4x32 on 32-bit words held in int64 (products wrap at 64 bits)"""
    low = 0xFFFFFFFF
    a, b = c0 * 0xD2511F53, c2 * 0xCD9E8D57
    return ((b >> 32) & low) ^ c1 ^ k0, b & low, ((a >> 32) & low) ^ c3 ^ k1, a & low


def _keep(n, d, p, seed, step, dev):
    """[n, d] truth values: which elements stay"""
    low = 0xFFFFFFFF
    c = torch.arange(-(-n * d // 4), device=dev)
    c0, c1, k0, k1 = c & low, c >> 32, seed & low, seed >> 32
    c2, c3 = torch.full_like(c, step & low), torch.full_like(c, step >> 32)
    for i in range(7):
        c0, c1, c2, c3 = _round(c0, c1, c2, c3, (k0 + i * 0x9E3779B9) & low, (k1 + i * 0xBB67AE85) & low)
    border = round(p * 2 ** 32)
    return torch.stack([c0 >= border, c1 >= border, c2 >= border, c3 >= border], 1).view(-1)[:n * d].view(n, d)


def _plain(s):
    case = s["case"]
    n, d, p, kind = case["rows"], case["dim"], case["p"], TYPES[case["dtype"]]
    x = s["x"].float()
    w, b = s["w"], s["b"]
    if case["op"] == "dropout":
        z = x if b is None else x + b
    else:
        v = x - x.mean(1, keepdim=True)
        rstd = 1.0 / torch.sqrt((v * v).mean(1, keepdim=True) + EPS)
        h = v * rstd
        z = h * w + b
    a = torch.where(z > 0, z, torch.zeros_like(z)) if case["relu"] else z
    keep = _keep(n, d, p, s["seed"], s["step"], x.device) if p > 0 else None
    scale = 1.0 / (1.0 - p)
    y = (a if keep is None else torch.where(keep, a * scale, torch.zeros_like(a))).to(kind)
    if case["pass"] == "forward":
        return {"y": y}
    dz = s["dy"].float()
    if keep is not None:
        dz = torch.where(keep, dz * scale, torch.zeros_like(dz))
    if case["relu"]:
        dz = torch.where(z > 0, dz, torch.zeros_like(dz))
    out = {"y": y}
    if case["op"] == "dropout":
        out["dx"] = dz.to(kind)
    else:
        g = dz * w
        out["dx"] = (rstd * (g - g.mean(1, keepdim=True) - h * (g * h).mean(1, keepdim=True))).to(kind)
        out["dw"] = (dz * h).sum(0)
    if b is not None:
        out["db"] = dz.sum(0)
    return out


def run(s):
    if not own:
        with torch.no_grad():
            return _plain(s)
    from artifact_b200 import norm
    case = s["case"]
    more = {} if case["p"] == 0 else {"p": case["p"], "seed": s["seed"], "step": s["step"]}
    with torch.set_grad_enabled(case["pass"] == "train"):
        if case["op"] == "dropout":
            y = norm.dropout(s["x"], bias=s["b"], relu=case["relu"], **more)
        else:
            y = norm.layer_norm(s["x"], s["w"], s["b"], EPS, relu=case["relu"], **more)
    if case["pass"] == "forward":
        return {"y": y}
    leaves = [(k, s[v]) for k, v in (("dx", "x"), ("dw", "w"), ("db", "b")) if s[v] is not None]
    grads = torch.autograd.grad(y, [t for _, t in leaves], s["dy"])
    return {"y": y.detach(), **{k: g for (k, _), g in zip(leaves, grads)}}


def work(case):
    n, d = case["rows"], case["dim"]
    e = n * d
    size = 4 if case["dtype"] == "f32" else 2
    train = case["pass"] == "train"
    vectors = 2 if case["op"] != "dropout" else int(case["bias"])
    # x in, y out; for training dy in and dx out; the vectors in, their gradients out
    moved = e * size * (4 if train else 2) + 4 * d * vectors * (2 if train else 1)
    per = {"norm": (8, 13), "dropout": (2, 2), "hidden": (10, 16)}[case["op"]]
    if case["p"] > 0:
        per = (per[0] + 14, per[1])                         # 56 integer operations for four elements, once
    return {"bytes": moved, "flops": e * (per[0] + (per[1] if train else 0))}


# ---- 64 bits ------------------------------------------------------------------------------------
def _stays(first, count, p, seed, step, dev):
    """which of the elements [first, first + count) stay; the 64-bit products from 16-bit halves"""
    e = torch.arange(first, first + count, device=dev)
    mask = (1 << 32) - 1

    def wide(m, v):
        ll = (m & 0xFFFF) * v                                # < 2^48
        hh = (m >> 16) * v + (ll >> 16)                      # < 2^49
        return hh >> 16, ((hh & 0xFFFF) << 16) | (ll & 0xFFFF)

    g = e // 4
    ctr = [g & mask, g >> 32, torch.zeros_like(g) + (step & mask), torch.zeros_like(g) + (step >> 32)]
    key = [seed & mask, seed >> 32]
    for _ in range(7):
        h0, l0 = wide(0xD2511F53, ctr[0])
        h1, l1 = wide(0xCD9E8D57, ctr[2])
        ctr = [h1 ^ ctr[1] ^ key[0], l1, h0 ^ ctr[3] ^ key[1], l0]
        key = [(key[0] + 0x9E3779B9) & mask, (key[1] + 0xBB67AE85) & mask]
    return torch.stack(ctr, 0).gather(0, (e % 4)[None])[0] >= round(p * 4294967296.0)


def exact(case, seed):
    s = prepare(case, seed)
    n, d, p = case["rows"], case["dim"], case["p"]
    dev = s["x"].device
    normed, train = case["op"] != "dropout", case["pass"] == "train"
    ys, dxs = [], []
    dw = torch.zeros(d, dtype=torch.float64, device=dev)
    db = torch.zeros_like(dw)
    step = max(1, (1 << 25) // d)
    for i in range(0, n, step):
        x = s["x"][i:i + step].detach().double().requires_grad_(train)
        w = s["w"].detach().double().requires_grad_(train) if normed else None
        b = s["b"].detach().double().requires_grad_(train) if s["b"] is not None else None
        z = x
        if normed:
            z = (x - x.sum(1, keepdim=True) / d) * (x.var(1, correction=0, keepdim=True) + EPS).rsqrt() * w
        if b is not None:
            z = z + b
        if case["relu"]:
            z = z * (z.detach() > 0)
        if p > 0:
            z = z * (_stays(i * d, x.shape[0] * d, p, s["seed"], s["step"], dev).view_as(z) / (1.0 - p))
        ys.append(z.detach())
        if train:
            z.backward(s["dy"][i:i + step].double())
            dxs.append(x.grad)
            dw += w.grad if w is not None else 0
            db += b.grad if b is not None else 0
    out = {"y": torch.cat(ys)}
    if train:
        out["dx"] = torch.cat(dxs)
        if normed:
            out["dw"] = dw
        if s["b"] is not None:
            out["db"] = db
    return out
