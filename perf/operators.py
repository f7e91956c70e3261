"""Performance cases of the feed-forward operators: what an adapted transformer block runs around its attention.

A case is one pass through one operator, as a training step or a sampler calls it:

* ``dropout``  ``dropout_add``: residual + dropout(x), its mask made again in the backward from a counter;
* ``gated``    ``gated_linear``: dropout(value * act(gate)), value and gate the two halves of one projection;
* ``linear``   ``linear_dropout_add``: residual + dropout(x W^T + b), the block's way back to its width.

With ``train`` a pass is the forward and the backward, and returns the output and every gradient; without, the
forward alone.

The random bits are those of Philox4x32-10 (Salmon et al., "Parallel random numbers: as easy as 1, 2, 3", 2011): element
(row, col) of the dropped matrix takes 16 bits of the block whose counter is (col // 8, row, offset low, offset high) and
whose key is the seed: half-word col % 8 of it, low halves first.  It is kept where those are at least
round(p * 65536), and divided by the share that is kept.
"""

import math

import numpy as np
import torch

own = False

DEVICE = "cuda"
DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
ACTIVATIONS = ("gelu", "gelu_tanh", "silu")


def listed():
    return [
        # The middle block of a small batch, one image's 64 places: a call that is all latency.
        dict(name="dropout_64x1280", kind="dropout", rows=64, cols=1280, dtype="bfloat16", p=0.1, residual=True, train=True),
        # A ragged matrix in the adapters' own type: rows that begin anywhere.
        dict(name="dropout_1111x333_f32", kind="dropout", rows=1111, cols=333, dtype="float32", p=0.25, residual=True, train=True),
        # The widest activations of a large batch: as much as the memory moves.
        dict(name="dropout_32768x2560", kind="dropout", rows=32768, cols=2560, dtype="bfloat16", p=0.1, residual=False, train=True),
        # One token through the widest block: the weights are read once and little is computed.
        dict(name="gated_token_1280", kind="gated", rows=1, d=1280, f=5120, dtype="bfloat16", act="gelu", p=0.0, bias=True, train=False),
        # A few tokens of a middle block in half precision, as a sampler steps a short batch.
        dict(name="gated_13_640_f16", kind="gated", rows=13, d=640, f=2560, dtype="float16", act="gelu", p=0.0, bias=True, train=False),
        # Odd sizes throughout, 32 bits: no row but the first is aligned.
        dict(name="gated_1001_333_f32", kind="gated", rows=1001, d=333, f=777, dtype="float32", act="silu", p=0.1, bias=True, train=True),
        # The narrow blocks at full resolution: four images of 64 x 64 places; short products, long outputs.
        dict(name="gated_16384_320", kind="gated", rows=16384, d=320, f=1280, dtype="bfloat16", act="gelu", p=0.1, bias=True, train=True),
        # The wide blocks over a large batch: 32 images of 16 x 16 places; the most work.
        dict(name="gated_8192_1280", kind="gated", rows=8192, d=1280, f=5120, dtype="bfloat16", act="gelu", p=0.0, bias=True, train=True),
        # The middle widths in the adapters' default type, 32 bits.
        dict(name="gated_4096_640_f32", kind="gated", rows=4096, d=640, f=2560, dtype="float32", act="gelu_tanh", p=0.0, bias=True, train=True),
        # One token back to the block's width.
        dict(name="linear_token_5120", kind="linear", rows=1, d=5120, n=1280, dtype="bfloat16", p=0.0, residual=True, bias=True, train=False),
        # A ragged batch in half precision.
        dict(name="linear_1025_2560_f16", kind="linear", rows=1025, d=2560, n=640, dtype="float16", p=0.1, residual=True, bias=True, train=True),
        # The wide blocks' way back over a large batch.
        dict(name="linear_8192_5120", kind="linear", rows=8192, d=5120, n=1280, dtype="bfloat16", p=0.1, residual=True, bias=True, train=True),
    ]


def draw(rng):
    def spread(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    def width(lo, hi):  # mostly multiples of 64, as models have them; any size now and then
        w = spread(lo, hi)
        return max(lo, (w + 32) // 64 * 64) if rng.random() < 0.7 else w

    kind = rng.choice(("dropout", "gated", "gated", "linear"))
    c = dict(kind=kind, dtype=rng.choice(("bfloat16", "bfloat16", "float16", "float32")), train=rng.random() < 0.7)
    c["p"] = round(rng.uniform(0.05, 0.5), 2) if c["train"] and (kind == "dropout" or rng.random() < 0.5) else 0.0
    if kind == "dropout":
        c["cols"], c["residual"], c["train"] = spread(64, 5120), rng.random() < 0.5, True
        c["rows"] = spread(1, 32768 * 2560 // c["cols"])
        c["p"] = c["p"] or 0.1
        return c
    most = 8192 * 1280 * 5120  # multiply-adds of the largest listed product
    if c["dtype"] == "float32":
        most //= 6
    c["bias"] = rng.random() < 0.8
    if kind == "gated":
        c["d"], c["f"], c["act"] = width(64, 1280), width(64, 5120), rng.choice(ACTIVATIONS)
        limit = min(16384, most // (c["d"] * c["f"]))
    else:
        c["d"], c["n"], c["residual"] = width(64, 5120), width(64, 1280), rng.random() < 0.5
        limit = min(16384, most // (c["d"] * c["n"]))
    c["rows"] = spread(1, limit) if c["train"] or rng.random() < 0.5 else spread(1, min(64, limit))
    return c


# ------------------------------------------------------------------------------------- inputs


def _widths(case):
    """(columns of x, columns of the output, rows of the weight)."""
    if case["kind"] == "dropout":
        return case["cols"], case["cols"], 0
    if case["kind"] == "gated":
        return case["d"], case["f"], 2 * case["f"]
    return case["d"], case["n"], case["n"]


def prepare(case, seed):
    g = torch.Generator(device=DEVICE).manual_seed(seed)
    dt = DTYPES[case["dtype"]]
    d_in, d_out, w_rows = _widths(case)
    rows = case["rows"]

    def normal(*shape, std=1.0):
        return (torch.randn(*shape, generator=g, device=DEVICE) * std).to(dt)

    s = {"case": case, "seed": (seed * 0x9E3779B97F4A7C15 + 12345) % 2 ** 63, "offset": seed % 1000 + 2 ** 33}
    s["x"] = normal(rows, d_in)  # what a norm gives
    s["residual"] = normal(rows, d_out, std=2.0) if case.get("residual") else None
    s["weight"] = normal(w_rows, d_in, std=d_in ** -0.5) if w_rows else None
    s["bias"] = normal(w_rows, std=0.1) if case.get("bias") else None
    if case["train"]:
        s["grad"] = normal(rows, d_out, std=1e-2)
        s["inputs"] = [s[k].requires_grad_(True) for k in ("x", "weight", "bias", "residual") if s[k] is not None]
    return s


def work(case):
    d_in, d_out, w_rows = _widths(case)
    rows, size = case["rows"], 4 if case["dtype"] == "float32" else 2
    x, y, w = rows * d_in, rows * d_out, w_rows * d_in
    b = w_rows if case.get("bias") else 0
    r = y if case.get("residual") else 0
    elements = x + w + b + r + y
    products = 1
    if case["train"]:
        elements += y + x + w + b  # the output's gradient is the residual's too
        products = 3
    # 30 operations for an element's random bits, 20 for an activation and as many for its derivative
    per = (30 if case["p"] else 0) + (20 if case["kind"] == "gated" else 1)
    return {"bytes": elements * size, "flops": products * 2 * rows * d_in * w_rows + y * per * (2 if case["train"] else 1)}


# --------------------------------------------------------------------------------- plain form


def _philox_keep(rows, cols, p, seed, offset):
    """[rows, cols] booleans: the elements that are kept."""
    n = (cols + 7) // 8
    c0 = torch.arange(n, device=DEVICE).expand(rows, n)
    c1 = torch.arange(rows, device=DEVICE)[:, None].expand(rows, n)
    c2, c3 = (torch.full((), v, dtype=torch.int64, device=DEVICE) for v in (offset & 0xFFFFFFFF, offset >> 32))
    k0, k1 = seed & 0xFFFFFFFF, seed >> 32

    def product(a, b):  # the high and the low 32 bits of a * b, in 16-bit steps that 63 bits hold
        low = a * (b & 0xFFFF)
        up = a * (b >> 16) + (low >> 16)
        return up >> 16, (up & 0xFFFF) << 16 | low & 0xFFFF

    for _ in range(10):
        h0, l0 = product(0xD2511F53, c0)
        h1, l1 = product(0xCD9E8D57, c2)
        c0, c1, c2, c3 = h1 ^ c1 ^ k0, l1, h0 ^ c3 ^ k1, l0
        k0, k1 = (k0 + 0x9E3779B9) & 0xFFFFFFFF, (k1 + 0xBB67AE85) & 0xFFFFFFFF
    words = torch.stack([c.expand(rows, n) for c in (c0, c1, c2, c3)], dim=-1)
    halves = torch.stack((words & 0xFFFF, words >> 16), dim=-1).reshape(rows, n * 8)[:, :cols]
    return halves >= _threshold(p)


def _threshold(p):
    return min(math.floor(p * 65536 + 0.5), 65536)


def _dropped(t, state):
    """t with its dropped elements zero and the others divided by the share that is kept."""
    case = state["case"]
    if case["p"] == 0:
        return t
    if "keep" not in state["pass"]:
        state["pass"]["keep"] = _philox_keep(*t.shape, case["p"], state["seed"], state["offset"])
    return torch.where(state["pass"]["keep"], t * (65536 / (65536 - _threshold(case["p"]))), 0.0)


def _activation(g, act):
    """act(g) and its derivative."""
    if act == "silu":
        s = 1 / (1 + torch.exp(-g))
        return g * s, s * (1 + g * (1 - s))
    if act == "gelu":
        cdf = 0.5 * (1 + torch.erf(g * math.sqrt(0.5)))
        return g * cdf, cdf + g * torch.exp(-0.5 * g * g) * (1 / math.sqrt(2 * math.pi))
    a, b = math.sqrt(2 / math.pi), 0.044715
    t = torch.tanh(a * (g + b * g * g * g))
    return 0.5 * g * (1 + t), 0.5 * (1 + t) + 0.5 * g * (1 - t * t) * a * (1 + 3 * b * g * g)


def _run_plain(state):
    case, dt = state["case"], DTYPES[state["case"]["dtype"]]
    state = dict(state)
    state["pass"] = {}  # what this pass alone keeps
    x, w, b, r, dy = (None if state.get(k) is None else state[k].detach().float() for k in ("x", "weight", "bias", "residual", "grad"))
    grads = []
    if case["kind"] == "dropout":
        y = _dropped(x, state)
        if case["train"]:
            grads = [_dropped(dy, state)]
    else:
        z = x @ w.t()
        if b is not None:
            z = z + b
        if case["kind"] == "gated":
            value, gate = z[:, :case["f"]], z[:, case["f"]:]
            a, slope = _activation(gate, case["act"])
            y = _dropped(value * a, state)
        else:
            y = _dropped(z, state)
        if case["train"]:
            dz = _dropped(dy, state)
            if case["kind"] == "gated":
                dz = torch.cat((dz * a, dz * value * slope), dim=1)
            grads = [dz @ w, dz.t() @ x] + ([dz.sum(0)] if b is not None else [])
    if r is not None:
        y = y + r
        if case["train"]:
            grads.append(dy)
    return [t.to(dt) for t in [y] + grads]


def run(state):
    if not own:
        with torch.no_grad():
            return _run_plain(state)
    from guass_amd.feedforward import dropout_add, gated_linear, linear_dropout_add

    case = state["case"]
    rng = dict(p=case["p"], seed=state["seed"], offset=state["offset"])

    def forward():
        if case["kind"] == "dropout":
            return dropout_add(state["x"], state["residual"], **rng)
        if case["kind"] == "gated":
            return gated_linear(state["x"], state["weight"], state["bias"], activation=case["act"], **rng)
        return linear_dropout_add(state["x"], state["weight"], state["bias"], state["residual"], **rng)

    if not case["train"]:
        with torch.no_grad():
            return [forward()]
    y = forward()
    return [y.detach(), *torch.autograd.grad(y, state["inputs"], state["grad"])]


# ------------------------------------------------------------------------------------ 64 bits


def _keep_words(rows, cols, p, seed, offset):
    """The kept elements, from 64-bit words on the host."""
    n = -(-cols // 8)
    mask = np.uint64(0xFFFFFFFF)
    ctr = [np.tile(np.arange(n, dtype=np.uint64), rows), np.repeat(np.arange(rows, dtype=np.uint64), n),
           np.full(rows * n, offset % 2 ** 32, np.uint64), np.full(rows * n, offset // 2 ** 32, np.uint64)]
    key = [seed % 2 ** 32, seed // 2 ** 32]
    s32 = np.uint64(32)
    for _ in range(10):
        a, b = ctr[0] * np.uint64(0xD2511F53), ctr[2] * np.uint64(0xCD9E8D57)  # below 2^64: exact
        ctr = [(b >> s32) ^ ctr[1] ^ np.uint64(key[0]), b & mask, (a >> s32) ^ ctr[3] ^ np.uint64(key[1]), a & mask]
        key = [(key[0] + 0x9E3779B9) % 2 ** 32, (key[1] + 0xBB67AE85) % 2 ** 32]
    bits = np.empty((rows * n, 4), dtype="<u4")
    for i, c in enumerate(ctr):
        bits[:, i] = c
    return torch.from_numpy(bits.view("<u2").reshape(rows, n * 8)[:, :cols] >= round(p * 65536)).to(DEVICE)


def exact(case, seed):
    s = prepare(case, seed)
    f64 = torch.float64
    x, w, b, r, dy = (None if s.get(k) is None else s[k].detach().to(f64) for k in ("x", "weight", "bias", "residual", "grad"))
    rows, d_out = case["rows"], _widths(case)[1]
    factor = 1.0
    if case["p"]:
        kept = 1 - round(case["p"] * 65536) / 65536
        factor = _keep_words(rows, d_out, case["p"], s["seed"], s["offset"]).to(f64) / kept
    if case["kind"] == "dropout":
        out = [x * factor] + ([dy * factor] if case["train"] else [])
    elif case["kind"] == "linear":
        out = [(torch.matmul(x, w.t()) + (0 if b is None else b)) * factor]
        if case["train"]:
            dz = dy * factor
            out += [torch.matmul(dz, w), torch.matmul(dz.t(), x)] + ([] if b is None else [dz.sum(0)])
    else:
        f = case["f"]
        value, gate = (torch.matmul(x, w[i * f:(i + 1) * f].t()) + (0 if b is None else b[i * f:(i + 1) * f]) for i in (0, 1))
        if case["act"] == "silu":  # g sigma(g), sigma' = sigma (1 - sigma)
            sig = torch.sigmoid(gate)
            act, slope = gate * sig, sig + gate * sig * (1 - sig)
        elif case["act"] == "gelu":  # g Phi(g), Phi' = phi
            cdf = torch.special.erfc(-gate / math.sqrt(2)) / 2
            act, slope = gate * cdf, cdf + gate * torch.exp(-gate ** 2 / 2) / math.sqrt(2 * math.pi)
        else:  # (1 + tanh u) / 2 = sigma(2u)
            sig = torch.sigmoid(2 * math.sqrt(2 / math.pi) * (gate + 0.044715 * gate ** 3))
            act = gate * sig
            slope = sig + gate * sig * (1 - sig) * 2 * math.sqrt(2 / math.pi) * (1 + 3 * 0.044715 * gate ** 2)
        out = [value * act * factor]
        if case["train"]:
            dv, dg = dy * factor * act, dy * factor * value * slope
            out += [torch.matmul(dv, w[:f]) + torch.matmul(dg, w[f:]), torch.cat((torch.matmul(dv.t(), x), torch.matmul(dg.t(), x)))]
            out += [] if b is None else [torch.cat((dv.sum(0), dg.sum(0)))]
    if r is not None:
        out[0] = out[0] + r
        if case["train"]:
            out.append(dy)
    return out
