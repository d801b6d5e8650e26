"""What the token operators are measured on (yolopoint_amd.utils.token_ops): layer norm with its backward pass, the fused
dropout + residual + layer norm, dropout from a counter-based generator, and rotary positions.

A token is a row of features: a keypoint's descriptor, a cell of the descriptor map, an entry of a sequence.  `run` makes one pass through an
operator -- the plain form in elementary torch operations, or the library's entry points where `own` is set.  `exact` is the definition in
64 bits.

Definitions shared by all of them:
  dropout     element i (flat, row-major) is kept where its 16 random bits are >= t = round(65536 p); kept values are multiplied by the fp32
              number nearest to 65536 / (65536 - t).  The bits: half i % 8 of the four words Philox4x32-10 gives for the counter
              (i / 8 [64 bits], offset [64 bits]) under the key `seed` [64 bits]; low halves first.
  fused sum   z = residual + dropout(x), rounded once to the type; y = layer_norm(z) of the rounded z.
  rotary      pair j of a head turns by positions[axis(j)] * inv_freq[j]; cos and sin are multiplied by `scale`.
"""
import math

import numpy as np
import torch

own = False

_TYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}


# ------------------------------------------------------------------------------------------------------------------ the cases
def _norm(rows, width, dtype, train, weights="f32"):
    return {"op": "layer_norm", "rows": rows, "width": width, "dtype": dtype, "train": train, "weights": weights}


def _fused(rows, width, dtype, train, p, weights="f32"):
    return {"op": "dropout_add_layer_norm", "rows": rows, "width": width, "dtype": dtype, "train": train, "p": p, "weights": weights}


def _dropout(rows, width, dtype, train, p, residual):
    return {"op": "dropout", "rows": rows, "width": width, "dtype": dtype, "train": train, "p": p, "residual": residual}


def _rotary(batch, tokens, q_heads, k_heads, head, rot, dtype, train, layout="bthd", interleaved=False, axes=1, base=10000.0, stretch=1.0, far=0):
    return {"op": "rotary", "batch": batch, "tokens": tokens, "q_heads": q_heads, "k_heads": k_heads, "head": head, "rot": rot, "dtype": dtype,
            "train": train, "layout": layout, "interleaved": interleaved, "axes": axes, "base": base, "stretch": stretch, "far": far}


def listed():
    return [
        # one token of the 256-wide descriptor on its way through a served block: nothing but latency
        dict(_norm(1, 256, "bf16", False), name="norm_one_token"),
        # the keypoints (1000 a frame) of a batch of 8 frames, a training step's pass
        dict(_norm(8 * 1000, 256, "bf16", True), name="norm_train_keypoints"),
        # tokens of a wide block, forward only (a long prompt, an evaluation)
        dict(_norm(16384, 4096, "f16", False, "same"), name="norm_wide_forward"),
        # odd rows and an odd width in fp32: no row but the first starts on a 16-byte border
        dict(_norm(5003, 1001, "f32", True), name="norm_train_odd_f32"),
        # a served block's residual + norm for the single tokens of 32 requests
        dict(_fused(32, 1024, "f16", False, 0.0, "same"), name="add_norm_served"),
        # a training step of an ordinary block over 8 x 1024 tokens
        dict(_fused(8 * 1024, 1024, "bf16", True, 0.1), name="fused_train_1024"),
        # every cell (80 x 80) of the descriptor maps of 64 images at 640 x 640, 256 features: the largest
        dict(_fused(64 * 6400, 256, "bf16", True, 0.1), name="fused_train_cells"),
        # dropout on a block's hidden layer, forward and gradient
        dict(_dropout(8 * 1024, 4096, "f16", True, 0.2, False), name="dropout_train_hidden"),
        # dropout into the residual, odd sizes, fp32
        dict(_dropout(3 * 1001, 777, "f32", True, 0.1, True), name="dropout_residual_odd"),
        # the next token of 64 requests, far into their contexts; half of the head turns
        dict(_rotary(64, 1, 32, 8, 128, 64, "bf16", False, stretch=4.0, far=131072), name="rotary_next_token"),
        # a training batch of long sequences, shared key heads, forward and gradient
        dict(_rotary(4, 8192, 16, 4, 128, 128, "bf16", True), name="rotary_train_long"),
        # keypoints at (x, y) in pixels, half of the head's pairs turned by each, heads in front of the tokens
        dict(_rotary(8, 1000, 4, 4, 64, 64, "f32", True, layout="bhtd", interleaved=True, axes=2, base=100.0), name="rotary_keypoints_2d"),
    ]


def _spread(rng, low, high):
    """A whole number between low and high, even over its logarithm."""
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def _wide(rng, low, high):
    """A width: a multiple of 64, of 8, or any number."""
    n = _spread(rng, low, high)
    step = rng.choice((64, 64, 8, 1))
    return max(low, n // step * step)


def draw(rng):
    op = rng.choice(("layer_norm", "layer_norm", "dropout_add_layer_norm", "dropout_add_layer_norm", "dropout", "rotary", "rotary"))
    dtype, train = rng.choice(("bf16", "bf16", "f16", "f32")), rng.random() < 0.6
    if op == "rotary":
        head = rng.choice((32, 64, 64, 80, 96, 128, 128, 256))
        axes = rng.choice((1, 1, 2))
        rot = rng.choice((head, head, head // 2))
        kv = rng.choice((1, 2, 4, 8))
        heads = kv * rng.choice((1, 1, 2, 4, 8))
        k_heads = rng.choice((kv, kv, 0))
        room = (96 << 20) // ((heads + kv) * head * (2 if dtype == "f32" else 1))
        tokens = 1 if rng.random() < 0.25 else _spread(rng, 2, min(32768, room))
        batch = _spread(rng, 1, min(128, max(1, room // tokens)))
        far = 0 if axes == 2 else rng.choice((0, 0, 4096, 1000000))
        return _rotary(batch, tokens, heads, k_heads, head, rot, dtype, train, rng.choice(("bthd", "bhtd")), rng.random() < 0.4, axes,
                       rng.choice((100.0, 10000.0, 500000.0)), rng.choice((1.0, 1.0, 8.0)), far)
    width = _wide(rng, 16, 8192)
    rows = _spread(rng, 1, max(1, min(262144, (96 << 20) // width // (2 if dtype == "f32" else 1))))
    weights = rng.choice(("f32", "same"))
    if op == "layer_norm":
        return _norm(rows, width, dtype, train, weights)
    if op == "dropout":
        return _dropout(rows, width, dtype, train, rng.choice((0.05, 0.1, 0.3, 0.5)), rng.random() < 0.5)
    return _fused(rows, width, dtype, train, rng.choice((0.0, 0.1, 0.1, 0.25)) if train else 0.0, weights)


def work(case):
    """Every input read once and every output written once; about what the formulas multiply and add."""
    size = 4 if case["dtype"] == "f32" else 2
    passes = 2 if case["train"] else 1
    if case["op"] == "rotary":
        tokens = case["batch"] * case["tokens"]
        values = tokens * (case["q_heads"] + case["k_heads"]) * case["head"]
        turned = tokens * (case["q_heads"] + case["k_heads"]) * case["rot"]
        places = tokens * case["axes"] * (4 if case["axes"] == 2 else 8)
        return {"bytes": passes * 2 * values * size + places, "flops": passes * 3 * turned}
    values = case["rows"] * case["width"]
    if case["op"] == "dropout":
        return {"bytes": (passes * 2 + (1 if case["residual"] else 0)) * values * size, "flops": passes * 2 * values}
    of_weights = 4 * case["width"] * (4 if case["weights"] == "f32" else size) // (1 if case["train"] else 2)
    if case["op"] == "layer_norm":
        return {"bytes": passes * 2 * values * size + of_weights, "flops": (8 + (12 if case["train"] else 0)) * values}
    return {"bytes": passes * 4 * values * size + of_weights, "flops": (10 + (15 if case["train"] else 0)) * values}


# ------------------------------------------------------------------------------------------------------------------ the inputs
def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(int(seed))
    dt, train = _TYPES[case["dtype"]], case["train"]
    s = {"case": case}

    def normal(*shape):
        return torch.randn(shape, device=dev, generator=g)

    if case["op"] == "rotary":
        B, T, D, ax = case["batch"], case["tokens"], case["head"], case["axes"]
        pairs = case["rot"] // 2 // ax
        steps = torch.arange(pairs, device=dev, dtype=torch.float64) / pairs
        s["inv_freq"] = (case["base"] ** -steps / case["stretch"]).repeat(ax)       # the table a program keeps
        s["scale"] = 0.1 * math.log(case["stretch"]) + 1.0 if case["stretch"] > 1.0 else 1.0
        if ax == 2:                                                                 # keypoints of a 640 x 640 image, between the pixels too
            s["positions"] = torch.rand((B, T, 2), device=dev, generator=g) * 639.0
        else:
            start = torch.randint(0, case["far"] + 1, (B, 1), device=dev, generator=g)
            s["positions"] = start + torch.arange(T, device=dev)
        for name, heads in (("q", case["q_heads"]), ("k", case["k_heads"])):
            if heads:
                shape = (B, T, heads, D) if case["layout"] == "bthd" else (B, heads, T, D)
                s[name] = normal(*shape).to(dt).requires_grad_(train)
                if train:
                    s["d" + name] = normal(*shape).to(dt)
        return s
    N, D = case["rows"], case["width"]
    spread = 0.5 + torch.rand(D, device=dev, generator=g) + 6.0 * (torch.rand(D, device=dev, generator=g) < 0.01)   # a few loud features
    shift = 0.3 * normal(D)

    def tokens():
        return (normal(N, D) * spread + shift).to(dt)

    s["x"] = tokens().requires_grad_(train)
    if train:
        s["dy"] = normal(N, D).to(dt)
    if case["op"] != "layer_norm":
        s["rng"] = (int(torch.randint(0, 1 << 62, (), device=dev, generator=g)), int(seed) % 1000003)
        if case["op"] == "dropout_add_layer_norm" or case["residual"]:
            s["residual"] = tokens().requires_grad_(train)
    if case["op"] != "dropout":
        wt = torch.float32 if case["weights"] == "f32" else dt
        s["weight"] = (1.0 + 0.2 * normal(D)).to(wt).requires_grad_(train)
        s["bias"] = (0.1 * normal(D)).to(wt).requires_grad_(train)
        if train and case["op"] == "dropout_add_layer_norm":
            s["dz"] = normal(N, D).to(dt)
    return s


# ------------------------------------------------------------------------------------------------------------------ the plain forms
def _threshold(p):
    t = int(math.floor(p * 65536.0 + 0.5))
    return t, float(np.float32(65536.0 / (65536 - t))) if t < 65536 else 0.0


def _keep(shape, p, rng, dev):
    """Which elements of a tensor of this shape dropout keeps."""
    n = math.prod(shape)
    low = 0xFFFFFFFF
    c0 = torch.arange((n + 7) // 8, device=dev)
    c1, c2, c3 = c0 >> 32, torch.full_like(c0, rng[1] & low), torch.full_like(c0, rng[1] >> 32)
    c0 = c0 & low
    k0, k1 = rng[0] & low, rng[0] >> 32
    for _ in range(10):
        a, b = c0 * 0xD2511F53, c2 * 0xCD9E8D57             # (64-bit products: they wrap, their bits are right)
        c0, c1, c2, c3 = ((b >> 32) & low) ^ c1 ^ k0, b & low, ((a >> 32) & low) ^ c3 ^ k1, a & low
        k0, k1 = (k0 + 0x9E3779B9) & low, (k1 + 0xBB67AE85) & low
    halves = torch.stack([c0 & 0xFFFF, c0 >> 16, c1 & 0xFFFF, c1 >> 16, c2 & 0xFFFF, c2 >> 16, c3 & 0xFFFF, c3 >> 16], dim=1)
    return (halves.view(-1)[:n] >= _threshold(p)[0]).view(shape)


def _plain_norm(z, w, b):
    z = z.float()
    d = z - z.mean(-1, keepdim=True)
    r = torch.rsqrt((d * d).mean(-1, keepdim=True) + 1e-5)
    return d * r * w.float() + b.float(), d * r, r


def _plain_norm_backward(dy, xhat, r, w):
    dy = dy.float()
    h = dy * w.float()
    dz = r * (h - h.mean(-1, keepdim=True) - xhat * (h * xhat).mean(-1, keepdim=True))
    return dz, (dy * xhat).sum(0).to(w.dtype), dy.sum(0).to(w.dtype)


def _plain(s):
    c = s["case"]
    if c["op"] == "rotary":
        a = s["positions"].double().unsqueeze(-1)                                    # angles of far positions: 64 bits
        if c["axes"] == 2:
            n = s["inv_freq"].numel() // 2
            a = torch.cat([a[..., 0, :] * s["inv_freq"][:n], a[..., 1, :] * s["inv_freq"][n:]], -1)
        else:
            a = a * s["inv_freq"]
        a = a.unsqueeze(2 if c["layout"] == "bthd" else 1)
        cos, sin = (torch.cos(a) * s["scale"]).float(), (torch.sin(a) * s["scale"]).float()

        def turn(x, sin):
            x = x.detach()
            rot, R = x[..., :c["rot"]].float(), c["rot"]
            u, v = (rot[..., 0::2], rot[..., 1::2]) if c["interleaved"] else (rot[..., :R // 2], rot[..., R // 2:])
            u, v = u * cos - v * sin, v * cos + u * sin
            rot = torch.stack([u, v], -1).flatten(-2) if c["interleaved"] else torch.cat([u, v], -1)
            return torch.cat([rot.to(x.dtype), x[..., R:]], -1)

        out = {name: turn(s[name], sin) for name in ("q", "k") if name in s}
        if c["train"]:
            out.update({"d" + name: turn(s["d" + name], -sin) for name in ("q", "k") if name in s})
        return out
    x = s["x"].detach()
    dt = x.dtype
    if c["op"] == "layer_norm":
        y, xhat, r = _plain_norm(x, s["weight"].detach(), s["bias"].detach())
        out = {"y": y.to(dt)}
        if c["train"]:
            dx, dw, db = _plain_norm_backward(s["dy"], xhat, r, s["weight"].detach())
            out.update(dx=dx.to(dt), dweight=dw, dbias=db)
        return out
    if c["op"] == "dropout":
        keep, factor = _keep(x.shape, c["p"], s["rng"], x.device), _threshold(c["p"])[1]
        y = torch.where(keep, x.float() * factor, 0.0)
        if c["residual"]:
            y = y + s["residual"].detach().float()
        out = {"y": y.to(dt)}
        if c["train"]:
            out["dx"] = torch.where(keep, s["dy"].float() * factor, 0.0).to(dt)
            if c["residual"]:
                out["dresidual"] = s["dy"]
        return out
    factor = _threshold(c["p"])[1]
    z = x.double() * factor                                                          # z is rounded, then normalised: 64 bits next to a border
    if c["p"] > 0.0:
        keep = _keep(x.shape, c["p"], s["rng"], x.device)
        z = torch.where(keep, z, 0.0)
    z = (z + s["residual"].detach().double()).to(dt)
    y, xhat, r = _plain_norm(z, s["weight"].detach(), s["bias"].detach())
    out = {"y": y.to(dt), "z": z}
    if c["train"]:
        dz, dw, db = _plain_norm_backward(s["dy"], xhat, r, s["weight"].detach())
        dz = dz + s["dz"].float()
        dx = dz * factor
        if c["p"] > 0.0:
            dx = torch.where(keep, dx, 0.0)
        out.update(dx=dx.to(dt), dresidual=dz.to(dt), dweight=dw, dbias=db)
    return out


# ------------------------------------------------------------------------------------------------------------------ the library's
def _own(s):
    from yolopoint_amd.utils import token_ops as ops
    c = s["case"]
    if c["op"] == "rotary":
        k = s.get("k")
        got = ops.rotary(s["q"], s["positions"], s["inv_freq"], k=k, interleaved=c["interleaved"], layout=c["layout"], scale=s["scale"])
        if k is None:
            out = {"q": got}
            if c["train"]:
                out["dq"], = torch.autograd.grad(got, s["q"], s["dq"])
            return out
        out = {"q": got[0], "k": got[1]}
        if c["train"]:
            out["dq"], out["dk"] = torch.autograd.grad(got, (s["q"], k), (s["dq"], s["dk"]))
        return out
    if c["op"] == "layer_norm":
        out = {"y": ops.layer_norm(s["x"], s["weight"], s["bias"])}
        if c["train"]:
            out["dx"], out["dweight"], out["dbias"] = torch.autograd.grad(out["y"], (s["x"], s["weight"], s["bias"]), s["dy"])
        return out
    if c["op"] == "dropout":
        res = s.get("residual")
        out = {"y": ops.dropout(s["x"], c["p"], s["rng"], residual=res)}
        if c["train"] and res is not None:
            out["dx"], out["dresidual"] = torch.autograd.grad(out["y"], (s["x"], res), s["dy"])
        elif c["train"]:
            out["dx"], = torch.autograd.grad(out["y"], s["x"], s["dy"])
        return out
    y, z = ops.dropout_add_layer_norm(s["x"], s["residual"], s["weight"], s["bias"], p=c["p"], rng=s["rng"])
    out = {"y": y, "z": z}
    if c["train"]:
        leaves = (s["x"], s["residual"], s["weight"], s["bias"])
        out["dx"], out["dresidual"], out["dweight"], out["dbias"] = torch.autograd.grad((y, z), leaves, (s["dy"], s["dz"]))
    return out


def run(state):
    return _own(state) if own else _plain(state)


# ------------------------------------------------------------------------------------------------------------------ the definition in 64 bits
def _bits(n, rng):
    """The 16 random bits of elements 0 .. n - 1, by numpy's unsigned arithmetic."""
    u = np.uint64
    g = np.arange((n + 7) // 8, dtype=u)
    low, half = u(0xFFFFFFFF), u(32)
    ctr = [g & low, g >> half, np.broadcast_to(u(rng[1] & 0xFFFFFFFF), g.shape), np.broadcast_to(u(rng[1] >> 32), g.shape)]
    key = [rng[0] & 0xFFFFFFFF, rng[0] >> 32]
    for r in range(10):
        p0, p1 = u(0xD2511F53) * ctr[0], u(0xCD9E8D57) * ctr[2]
        ctr = [(p1 >> half) ^ ctr[1] ^ u(key[0]), p1 & low, (p0 >> half) ^ ctr[3] ^ u(key[1]), p0 & low]
        key = [(key[0] + 0x9E3779B9) % (1 << 32), (key[1] + 0xBB67AE85) % (1 << 32)]
    words = np.stack(ctr, axis=1).astype("<u4")
    return words.view("<u2").reshape(-1)[:n].astype(np.int32)


def exact(case, seed):
    s = prepare(case, seed)
    d = {k: v.detach().double() for k, v in s.items() if isinstance(v, torch.Tensor)}
    if case["op"] == "rotary":
        half, R = case["rot"] // 2, case["rot"]
        place = d["positions"] if case["axes"] == 2 else d["positions"].unsqueeze(-1)
        angle = place.repeat_interleave(half // case["axes"], dim=-1) * d["inv_freq"]
        angle = angle.unsqueeze(2) if case["layout"] == "bthd" else angle.unsqueeze(1)
        turn = torch.polar(torch.full_like(angle, s["scale"]), angle)
        index = torch.arange(R, device=angle.device)
        first, second = (index[0::2], index[1::2]) if case["interleaved"] else (index[:half], index[half:])

        def turned(x, by):
            w = torch.complex(x[..., first], x[..., second]) * by
            x = x.clone()
            x[..., first], x[..., second] = w.real, w.imag
            return x

        out = {n: turned(d[n], turn) for n in ("q", "k") if n in d}
        if case["train"]:
            out.update({"d" + n: turned(d["d" + n], turn.conj()) for n in ("q", "k") if n in d})
        return out
    N, D = case["rows"], case["width"]
    mask = None
    if case["op"] != "layer_norm":
        t = round(case["p"] * 65536)
        factor = float(np.float32(65536 / (65536 - t)))
        mask = factor
        if t:
            mask = torch.from_numpy(np.where(_bits(N * D, s["rng"]) < t, 0.0, factor).astype(np.float32)).to(d["x"].device).double().view(N, D)
    if case["op"] == "dropout":
        y = d["x"] * mask + (d["residual"] if case["residual"] else 0.0)
        out = {"y": y}
        if case["train"]:
            out["dx"] = d["dy"] * mask
            if case["residual"]:
                out["dresidual"] = d["dy"]
        return out
    z = d["x"]
    out = {}
    if case["op"] == "dropout_add_layer_norm":
        z = (z * mask + d["residual"]).to(_TYPES[case["dtype"]])                     # (the stored sum is what is normalised)
        out["z"] = z = z.double()
    var, mean = torch.var_mean(z, dim=-1, unbiased=False, keepdim=True)
    sigma = torch.sqrt(var + 1e-5)
    xhat = (z - mean) / sigma
    out["y"] = torch.addcmul(d["bias"], xhat, d["weight"])
    if case["train"]:
        a = d["dy"] * d["weight"]
        along = torch.einsum("nd,nd->n", a, xhat).unsqueeze(-1) / D
        dz = (a - a.sum(-1, keepdim=True) / D - along * xhat) / sigma
        out["dweight"], out["dbias"] = torch.einsum("nd,nd->d", d["dy"], xhat), d["dy"].sum(0)
        if case["op"] == "layer_norm":
            out["dx"] = dz
        else:
            dz = dz + d["dz"]
            out["dresidual"], out["dx"] = dz, dz * mask
    return out
