"""Cases of the learned-appearance operators (tidegs_b200.appearance): layer
norm, gated feed-forward block and counter-based dropout over the rows of the
resident Gaussians, for rendering (forward) and for training (forward and
backward).

`own` selects the framework's kernels; without it `run` computes the same
results from elementary torch operations in 32 bits.
"""
import math

import numpy as np
import torch

own = False

DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
SIZE = {"fp32": 4, "bf16": 2, "fp16": 2}
EPS = 1e-5
PARAMS = ("x", "weight", "bias", "w_gate", "w_up", "w_down")

# Largest work of one pass: bytes of the row operators, operations of the
# feed-forward block (a drawn case stays within these).
MOST_BYTES = 1.1e9
MOST_FLOPS = 4.2e11


def listed():
    return [
        # One small view of a scene: the call's latency.
        dict(name="norm_view", op="norm", train=False, n=1500, c=64, dtype="fp32"),
        # Features of 128 resident blocks of 16,384 Gaussians, rendered.
        dict(name="norm_blocks", op="norm", train=False, n=2097152, c=64, dtype="bf16"),
        # Whole 59-column Gaussian rows: an odd width, training.
        dict(name="norm_rows_train", op="norm", train=True, n=786432, c=59, dtype="fp32"),
        # Wide features of a coarse level of detail, training; ragged count.
        dict(name="norm_wide_train", op="norm", train=True, n=100003, c=768, dtype="bf16"),
        # A small view's colors.
        dict(name="ffn_view", op="ffn", train=False, n=1500, d=32, h=64, o=3, dtype="bf16"),
        # Residuals of the 16 x 3 SH coefficients of 128 resident blocks.
        dict(name="ffn_blocks", op="ffn", train=False, n=2097152, d=64, h=128, o=48, dtype="bf16"),
        # The same head in training, half the blocks.
        dict(name="ffn_blocks_train", op="ffn", train=True, n=1048576, d=64, h=128, o=48, dtype="bf16"),
        # Wide head over a ragged count of visible Gaussians, training.
        dict(name="ffn_wide_train", op="ffn", train=True, n=200001, d=128, h=384, o=128, dtype="bf16"),
        # Head kept in 32 bits, odd widths, training.
        dict(name="ffn_fp32_train", op="ffn", train=True, n=131071, d=35, h=96, o=3, dtype="fp32"),
        # Whole Gaussians dropped by their global ids (opacities), training.
        dict(name="dropout_opacity_train", op="dropout", train=True, n=4194304, c=1, per_row=True, ids=True,
             p=0.1, dtype="fp32"),
        # Appearance features dropped one by one, training.
        dict(name="dropout_features_train", op="dropout", train=True, n=1048576, c=64, per_row=False, ids=False,
             p=0.25, dtype="bf16"),
        # A view's features, odd width.
        dict(name="dropout_view_train", op="dropout", train=True, n=20011, c=27, per_row=False, ids=True, p=0.5,
             dtype="fp32"),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(("norm", "ffn", "ffn", "dropout"))
    case = dict(op=op, train=rng.random() < 0.6, n=_log(rng, 1, 2500000))
    if op == "norm":
        case |= dict(c=_log(rng, 3, 1024), dtype=rng.choice(("fp32", "bf16", "fp16")))
    elif op == "ffn":
        case |= dict(d=_log(rng, 8, 256), h=_log(rng, 16, 512), o=_log(rng, 3, 256),
                     dtype=rng.choice(("bf16", "bf16", "fp32")))
        if rng.random() < 0.5:  # most heads have widths of whole vectors
            case |= dict(d=-(-case["d"] // 16) * 16, h=-(-case["h"] // 16) * 16)
    else:
        case |= dict(c=_log(rng, 1, 256), per_row=rng.random() < 0.4, ids=rng.random() < 0.5,
                     p=rng.choice((0.05, 0.1, 0.25, 0.5, 0.9)), dtype=rng.choice(("fp32", "bf16", "fp16")))
    most = MOST_FLOPS / (8 if case["dtype"] == "fp32" else 1)
    w = work(case)
    over = max(w["flops"] / most, w["bytes"] / MOST_BYTES)
    if over > 1:
        case["n"] = max(1, int(case["n"] / over))
    return case


def work(case):
    n, s = case["n"], SIZE[case["dtype"]]
    if case["op"] == "norm":
        c = case["c"]
        # forward: x in, y out; training also the gradient in and out
        return dict(bytes=n * c * s * (4 if case["train"] else 2) + c * s * (4 if case["train"] else 2),
                    flops=n * c * (20 if case["train"] else 8))
    if case["op"] == "ffn":
        d, h, o = case["d"], case["h"], case["o"]
        weights = 2 * d * h + h * o
        if not case["train"]:
            return dict(bytes=s * (n * (d + o) + weights), flops=2 * n * weights)
        # training: x and the output's gradient in, the output and x's gradient out; three times the forward's products
        return dict(bytes=s * (n * (2 * d + 2 * o) + 2 * weights), flops=6 * n * weights)
    c = case["c"]
    passes = 4 if case["train"] else 2
    return dict(bytes=n * c * s * passes + (8 * n if case["ids"] else 0), flops=n * c * passes)


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def prepare(case, seed):
    g, n, t = _gen(seed), case["n"], DTYPES[case["dtype"]]

    def rand(*shape, scale=1.0):
        return (torch.randn(*shape, generator=g, device="cuda") * scale).to(t)

    s = dict(case=case, n=n)
    if case["op"] == "ffn":
        d, h, o = case["d"], case["h"], case["o"]
        s |= dict(x=rand(n, d), w_gate=rand(h, d, scale=d ** -0.5), w_up=rand(h, d, scale=d ** -0.5),
                  w_down=rand(o, h, scale=h ** -0.5))
        shape = (n, o)
    else:
        shape = (n, case["c"])
        x = torch.randn(*shape, generator=g, device="cuda")
        if case["op"] == "norm":  # rows of their own mean and spread
            x = x * (0.5 + torch.rand(n, 1, generator=g, device="cuda")) + torch.randn(n, 1, generator=g, device="cuda")
            s |= dict(weight=(1 + 0.1 * torch.randn(case["c"], generator=g, device="cuda")).to(t),
                      bias=rand(case["c"], scale=0.1))
        s |= dict(x=x.to(t))
    if case["op"] == "dropout":
        # the visible Gaussians' global ids: ascending, with gaps, past 32 bits
        s |= dict(seed=(int(seed) * 6364136223846793005 + 1) % (1 << 64), step=int(seed) % 1000 + 1, ids=None)
        if case["ids"]:
            s["ids"] = torch.cumsum(torch.randint(1, 4, (n,), generator=g, device="cuda"), 0) + ((1 << 32) - n)
    if case["train"]:
        # the renderer's gradients: small, and zero for the rows that no pixel saw
        seen = torch.rand(n, 1, generator=g, device="cuda") < 0.7
        s["grad"] = (torch.randn(*shape, generator=g, device="cuda") * 1e-3 * seen).to(t)
        for k in PARAMS:
            if k in s:
                s[k].requires_grad_(True)
    return s


def run(s):
    case = s["case"]
    if own:
        return _run_own(s, case)
    with torch.no_grad():
        return {"norm": _norm, "ffn": _ffn, "dropout": _dropout}[case["op"]](s, case)


def _run_own(s, case):
    from tidegs_b200 import appearance as ap

    def forward():
        if case["op"] == "norm":
            return ap.layer_norm(s["x"], s["weight"], s["bias"], EPS)
        if case["op"] == "ffn":
            return ap.gated_feed_forward(s["x"], s["w_gate"], s["w_up"], s["w_down"])
        return ap.dropout(s["x"], case["p"], s["seed"], offset=s["step"], ids=s["ids"], per_row=case["per_row"])

    if not case["train"]:
        with torch.no_grad():
            return dict(y=forward())
    y = forward()
    names = [k for k in PARAMS if k in s]
    grads = torch.autograd.grad(y, [s[k] for k in names], s["grad"])
    return dict(y=y.detach()) | {"grad_" + k: g for k, g in zip(names, grads)}


# --- plain forms -----------------------------------------------------------

def _norm(s, case):
    t = s["x"].dtype
    x, w, b = s["x"].float(), s["weight"].float(), s["bias"].float()
    x = x - x.mean(1, keepdim=True)
    rstd = torch.rsqrt((x * x).mean(1, keepdim=True) + EPS)
    xhat = x * rstd
    out = dict(y=(xhat * w + b).to(t))
    if case["train"]:
        dy = s["grad"].float()
        gy = dy * w
        dx = rstd * (gy - gy.mean(1, keepdim=True) - xhat * (gy * xhat).mean(1, keepdim=True))
        # sums over millions of rows in 64 bits
        out |= dict(grad_x=dx.to(t), grad_weight=(dy * xhat).sum(0, dtype=torch.float64).to(t),
                    grad_bias=dy.sum(0, dtype=torch.float64).to(t))
    return out


def _ffn(s, case):
    t = s["x"].dtype
    x, wg, wu, wd = (s[k].float() for k in ("x", "w_gate", "w_up", "w_down"))
    g, u = x @ wg.T, x @ wu.T
    sig = torch.sigmoid(g)
    a = g * sig
    h = a * u
    out = dict(y=(h @ wd.T).to(t))
    if case["train"]:
        dy = s["grad"].float()
        dh = dy @ wd
        du = dh * a
        dg = dh * u * sig * (1 + g * (1 - sig))
        out |= dict(grad_x=(dg @ wg + du @ wu).to(t), grad_w_gate=(dg.T @ x).to(t), grad_w_up=(du.T @ x).to(t),
                    grad_w_down=(dy.T @ h).to(t))
    return out


def _philox(c0, c1, c2, c3, seed):
    """Philox4x32-10 (Salmon, Moraes, Dror and Shaw, 2011) on int64 tensors of 32-bit words."""
    mask = 0xFFFFFFFF
    k0, k1 = seed & mask, (seed >> 32) & mask

    def mul(m, v):  # 32 x 32 -> high and low words, within signed 64 bits
        low = (v & 0xFFFF) * m
        high = (v >> 16) * m + (low >> 16)
        return high >> 16, ((high & 0xFFFF) << 16) | (low & 0xFFFF)

    for _ in range(10):
        h0, l0 = mul(0xD2511F53, c0)
        h1, l1 = mul(0xCD9E8D57, c2)
        c0, c1, c2, c3 = h1 ^ c1 ^ k0, l1, h0 ^ c3 ^ k1, l0
        k0, k1 = (k0 + 0x9E3779B9) & mask, (k1 + 0xBB67AE85) & mask
    return c0, c1, c2, c3


def _kept(s, case, n, c):
    ids = torch.arange(n, device="cuda") if s["ids"] is None else s["ids"]
    ids = ids[:, None]
    groups = torch.arange(1 if case["per_row"] else -(-c // 4), device="cuda")[None, :]
    shape = (n, groups.shape[1])
    words = _philox((ids & 0xFFFFFFFF).expand(shape), ((ids >> 32) & 0xFFFFFFFF).expand(shape), groups.expand(shape),
                    torch.full(shape, s["step"], device="cuda"), s["seed"])
    limit = int(case["p"] * 2 ** 32)
    if case["per_row"]:
        return words[0] >= limit
    return (torch.stack(words, 2) >= limit).reshape(n, -1)[:, :c]


def _dropout(s, case):
    x = s["x"]
    kept = _kept(s, case, *x.shape)
    scale = 1.0 / (1.0 - case["p"])
    zero = torch.zeros((), device="cuda")
    out = dict(y=torch.where(kept, x.float() * scale, zero).to(x.dtype))
    if case["train"]:
        out["grad_x"] = torch.where(kept, s["grad"].float() * scale, zero).to(x.dtype)
    return out


# --- from the definitions, in 64 bits ---------------------------------------

def _words(ids, groups, step, seed):
    """The four Philox4x32-10 words of every (id, group), as a numpy array [n, groups, 4]."""
    m = np.uint64(0xFFFFFFFF)
    b = np.uint64(32)
    ids = ids.astype(np.uint64)[:, None]
    c = [np.broadcast_to(v, (len(ids), groups)) for v in (ids & m, ids >> b, np.arange(groups, dtype=np.uint64)[None, :],
                                                         np.full((1, 1), step, np.uint64))]
    for r in range(10):
        k0, k1 = ((((seed >> s) & 0xFFFFFFFF) + r * w) & 0xFFFFFFFF for s, w in ((0, 0x9E3779B9), (32, 0xBB67AE85)))
        p, q = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        c = [(q >> b) ^ c[1] ^ np.uint64(k0), q & m, (p >> b) ^ c[3] ^ np.uint64(k1), p & m]
    return np.stack(c, 2)


def exact(case, seed):
    s = prepare(case, seed)
    x = s["x"].detach().double()
    dy = s["grad"].double() if case["train"] else None
    if case["op"] == "norm":
        w, b = s["weight"].detach().double(), s["bias"].detach().double()
        var, mean = torch.var_mean(x, dim=1, correction=0, keepdim=True)
        std = torch.sqrt(var + EPS)
        z = (x - mean) / std
        out = dict(y=torch.addcmul(b, z, w))
        if case["train"]:
            v = dy * w
            c = x.shape[1]
            out |= dict(grad_x=(v - (v.sum(1, keepdim=True) + z * torch.einsum("nc,nc->n", v, z)[:, None]) / c) / std,
                        grad_weight=torch.einsum("nc,nc->c", dy, z), grad_bias=dy.sum(0))
        return out
    if case["op"] == "ffn":
        wg, wu, wd = (s[k].detach().double().requires_grad_(case["train"]) for k in ("w_gate", "w_up", "w_down"))
        x.requires_grad_(case["train"])
        gate = x @ wg.T
        y = (gate / (1 + torch.exp(-gate)) * (x @ wu.T)) @ wd.T
        if not case["train"]:
            return dict(y=y)
        grads = torch.autograd.grad(y, (x, wg, wu, wd), dy)
        return dict(y=y.detach()) | dict(zip(("grad_x", "grad_w_gate", "grad_w_up", "grad_w_down"), grads))
    n, c = x.shape
    ids = np.arange(n) if s["ids"] is None else s["ids"].cpu().numpy()
    words = _words(ids, 1 if case["per_row"] else (c + 3) // 4, s["step"], s["seed"])
    words = words[:, 0, :1] if case["per_row"] else words.reshape(n, -1)[:, :c]
    kept = torch.from_numpy(words >= np.uint64(int(case["p"] * 2 ** 32))).cuda()
    out = dict(y=x * kept / (1 - case["p"]))
    if case["train"]:
        out["grad_x"] = dy * kept / (1 - case["p"])
    return out
