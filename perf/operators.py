"""Cases of the 8-bit operators: what they are given, their plain forms, the calls a user makes.

norm_q8      root-mean-square norm with the residual's addition, output in 8 bits with a scale per row (serving)
linear_q8    matrix product of 8-bit integers with a scale per token and per output channel (serving)
norm_ckpt    the norm with the residual's addition in training: forward, and a backward that reads an 8-bit checkpoint
weight_grad  a linear's input kept in 8 bits, and the weight gradient formed from what was kept

8-bit rows:        q = round(v * 127 / max|v|), v = (x + residual) * weight; the row stands for q * (max|v| * rstd / 127).
8-bit checkpoints: groups of 128 columns, each with the smallest power of two s (at least 2^-100) that keeps |v| / s <= 127;
                   q = round(v / s), kept value q * s.
"""
import math

import torch

own = False

EPS = 1e-5
GROUP = 128
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def listed():
    return [
        # one decoding step of eight sequences: the norm before in_proj at d_model 1024
        {"name": "norm_q8_step", "op": "norm_q8", "rows": 8, "cols": 1024, "dtype": "bf16"},
        # a long bf16 prefill at d_model 1024
        {"name": "norm_q8_long", "op": "norm_q8", "rows": 65536, "cols": 1024, "dtype": "bf16"},
        # one token through in_proj (d_model 1024, expand 2)
        {"name": "linear_step", "op": "linear_q8", "rows": 1, "inner": 1024, "outer": 4096, "dtype": "bf16", "bias": False},
        # a decoding batch through out_proj of the next size, with a bias
        {"name": "linear_batch", "op": "linear_q8", "rows": 48, "inner": 4096, "outer": 2048, "dtype": "bf16", "bias": True},
        # the classifier's in_proj over its whole batch: 256 sequences of 300 steps, d_model 256
        {"name": "linear_classifier", "op": "linear_q8", "rows": 76800, "inner": 256, "outer": 1024, "dtype": "f32", "bias": False},
        # a prefill in earnest: 16384 tokens through a wide projection
        {"name": "linear_prefill", "op": "linear_q8", "rows": 16384, "inner": 4096, "outer": 8192, "dtype": "bf16", "bias": False},
        # the four-layer stack's training step (batch 32, length 1024, d_model 128)
        {"name": "norm_ckpt_stack", "op": "norm_ckpt", "rows": 32768, "cols": 128, "dtype": "f32"},
        # a ragged batch at a width that no vector load divides
        {"name": "norm_ckpt_ragged", "op": "norm_ckpt", "rows": 2399, "cols": 1001, "dtype": "f16"},
        # a long bf16 sequence
        {"name": "norm_ckpt_long", "op": "norm_ckpt", "rows": 65536, "cols": 1024, "dtype": "bf16"},
        # in_proj's weight gradient in the four-layer stack, behind the norm
        {"name": "weight_grad_stack", "op": "weight_grad", "rows": 32768, "inner": 128, "outer": 512, "dtype": "f32", "normed": True},
        # odd sizes throughout
        {"name": "weight_grad_ragged", "op": "weight_grad", "rows": 4099, "inner": 333, "outer": 777, "dtype": "f16", "normed": False},
        # in_proj's weight gradient over a long bf16 sequence, behind the norm
        {"name": "weight_grad_long", "op": "weight_grad", "rows": 65536, "inner": 1024, "outer": 4096, "dtype": "bf16", "normed": True},
    ]


def draw(rng):
    def size(low, high):
        n = max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high + 1)))))))
        return n - 1 if n == 3072 else n

    def width(step):
        n = max(step, size(64, 8192) // step * step)
        return n + step if n == 3072 else n

    op = rng.choice(("norm_q8", "linear_q8", "norm_ckpt", "weight_grad"))
    case = {"op": op, "dtype": rng.choice(("f32", "bf16", "f16"))}
    if op in ("norm_q8", "norm_ckpt"):
        cols = width(1)
        case.update(rows=size(1, min(76800, (1 << 26) // cols // 2)), cols=cols)
        return case
    # widths in multiples of a vector, as models have them, or any at all
    step = rng.choice((1, 8, 64))
    inner, outer = width(step), width(step)
    if op == "linear_q8":
        rows = size(1, min(76800, (1 << 27) // outer, (1 << 38) // (inner * outer)))
        case.update(rows=rows, inner=inner, outer=outer, bias=rng.random() < 0.5)
    else:
        most = min(65536, (1 << 37) // (inner * outer), (1 << 27) // (inner + outer))
        case.update(rows=size(1, most), inner=inner, outer=outer, normed=rng.random() < 0.5)
    return case


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def _activations(g, rows, cols, dtype):
    """Normal activations whose channels differ in size, as a residual stream's do."""
    channel = torch.exp(0.5 * torch.randn(cols, generator=g, device="cuda"))
    return (torch.randn(rows, cols, generator=g, device="cuda") * channel).to(dtype)


def _rows8(g, rows, cols, std):
    """8-bit rows as quantising them leaves them: rows start on 16-byte boundaries, the largest value is 127."""
    pitch = (cols + 15) // 16 * 16
    q = torch.zeros(rows, pitch, dtype=torch.int8, device="cuda")[:, :cols]
    v = torch.randn(rows, cols, generator=g, device="cuda").clamp_(-4, 4)
    top = v.abs().amax(1, keepdim=True)
    q.copy_(torch.round(v * (127 / top)))
    return q, (top[:, 0] * (std / 127)).contiguous()


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    op, rows, dtype = case["op"], case["rows"], DTYPES[case["dtype"]]
    s = {"op": op, "dtype": dtype}
    if op == "linear_q8":
        s["xq"], s["xs"] = _rows8(g, rows, case["inner"], 1.0)
        s["wq"], s["ws"] = _rows8(g, case["outer"], case["inner"], case["inner"] ** -0.5)
        s["bias"] = torch.randn(case["outer"], generator=g, device="cuda") * 0.1 if case["bias"] else None
        return s
    if op == "weight_grad":
        s["x"] = _activations(g, rows, case["inner"], dtype)
        s["dy"] = torch.randn(rows, case["outer"], generator=g, device="cuda").to(dtype)
        s["rstd"] = s["w"] = None
        if case["normed"]:
            s["rstd"] = torch.rsqrt(s["x"].float().square().mean(1) + EPS)
            s["w"] = 1 + 0.1 * torch.randn(case["inner"], generator=g, device="cuda")
        return s
    cols = case["cols"]
    s["x"] = _activations(g, rows, cols, dtype)
    s["residual"] = _activations(g, rows, cols, dtype)
    s["w"] = 1 + 0.1 * torch.randn(cols, generator=g, device="cuda")
    if op == "norm_ckpt":
        s["dn"] = torch.randn(rows, cols, generator=g, device="cuda").to(dtype)
        s["dh"] = torch.randn(rows, cols, generator=g, device="cuda").to(dtype)
        for name in ("x", "residual", "w"):
            s[name].requires_grad_()
    return s


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------
def run(state):
    return (_own if own else _plain)(state)


def _own(s):
    from momentummamba_b200 import int8

    if s["op"] == "norm_q8":
        n, h = int8.rms_norm_q8(s["x"], s["w"], residual=s["residual"], eps=EPS)
        return {"n": n.dequantize(s["dtype"]), "h": h}
    if s["op"] == "linear_q8":
        return int8.linear_q8(int8.Q8Rows(s["xq"], s["xs"]), int8.Q8Rows(s["wq"], s["ws"]), s["bias"], out_dtype=s["dtype"])
    if s["op"] == "norm_ckpt":
        n, h = int8.rms_norm_ckpt(s["x"], s["w"], residual=s["residual"], eps=EPS)
        dx, dw = torch.autograd.grad([n, h], [s["x"], s["w"]], [s["dn"], s["dh"]])
        return {"n": n, "h": h, "dx": dx, "dw": dw}
    kept = int8.checkpoint_rows(s["x"])
    return int8.weight_grad_ckpt(s["dy"], kept, row_scale=s["rstd"], col_scale=s["w"])


def _kept(v):
    """What an 8-bit checkpoint of v (rows, cols) in 32 bits holds."""
    rows, cols = v.shape
    groups = -(-cols // GROUP)
    v = torch.nn.functional.pad(v, (0, groups * GROUP - cols)).view(rows, groups, GROUP)
    m, e = torch.frexp(v.abs().amax(2, keepdim=True))
    s = torch.ldexp(torch.ones_like(m), torch.clamp(torch.where(m * 128 > 127, e - 6, e - 7), min=-100))
    return (torch.round(v / s) * s).view(rows, -1)[:, :cols]


@torch.no_grad()
def _plain(s):
    if s["op"] == "linear_q8":
        y = (s["xq"].float() @ s["wq"].float().t()) * s["xs"][:, None] * s["ws"]
        return (y if s["bias"] is None else y + s["bias"]).to(s["dtype"])
    if s["op"] == "weight_grad":
        dy, kept = s["dy"].float(), _kept(s["x"].float())
        if s["rstd"] is None:
            return (dy.t() @ kept).to(s["dtype"])
        return ((dy * s["rstd"][:, None]).t() @ kept * s["w"]).to(s["dtype"])
    h, w = s["x"].float() + s["residual"].float(), s["w"]
    rstd = torch.rsqrt((h * h).mean(1, keepdim=True) + EPS)
    if s["op"] == "norm_q8":
        v = h * w
        top = v.abs().amax(1, keepdim=True)
        q = torch.round(v * torch.where(top > 0, 127 / top, 0.0))
        return {"n": (q * (top * rstd / 127)).to(s["dtype"]), "h": h.to(s["dtype"])}
    dn, n = s["dn"].float(), _kept(h) * rstd
    g = dn * w
    dx = rstd * (g - n * (g * n).mean(1, keepdim=True)) + s["dh"].float()
    return {"n": (h * rstd * w).to(s["dtype"]), "h": h.to(s["dtype"]), "dx": dx.to(s["dtype"]), "dw": (dn * n).sum(0)}


# ---------------------------------------------------------------------------
# what a pass cannot do without, and its values in 64 bits
# ---------------------------------------------------------------------------
def work(case):
    rows, e = case["rows"], DTYPES[case["dtype"]].itemsize
    if case["op"] == "linear_q8":
        k, n = case["inner"], case["outer"]
        return {"bytes": rows * k + n * k + 4 * (rows + n + (n if case["bias"] else 0)) + e * rows * n, "flops": 2 * rows * n * k}
    if case["op"] == "weight_grad":
        k, n = case["inner"], case["outer"]
        return {"bytes": e * (rows * (k + n) + n * k) + (4 * (rows + k) if case["normed"] else 0), "flops": 2 * rows * n * k}
    cols = case["cols"]
    if case["op"] == "norm_q8":  # x, residual in; the sum and the rows out
        return {"bytes": 4 * e * rows * cols + 4 * cols, "flops": 8 * rows * cols}
    # x, residual, both gradients in; the norm, the sum and dx out
    return {"bytes": 7 * e * rows * cols + 8 * cols, "flops": 20 * rows * cols}


def _kept64(v):
    rows, cols = v.shape
    out = torch.empty_like(v)
    for at in range(0, cols, GROUP):
        part = v[:, at:at + GROUP]
        top = part.abs().max(1).values
        step = torch.exp2(torch.floor(torch.log2(torch.where(top > 0, top, torch.ones_like(top)))) - 6)
        step = torch.where(top / step > 127, 2 * step, step).clamp(min=2.0 ** -100)[:, None]
        out[:, at:at + GROUP] = step * torch.round(part / step)
    return out


@torch.no_grad()
def exact(case, seed):
    s = prepare(case, seed)
    d = {k: v.double() for k, v in s.items() if isinstance(v, torch.Tensor)}
    if s["op"] == "linear_q8":
        y = torch.mm(d["xq"] * d["xs"].unsqueeze(1), (d["wq"] * d["ws"].unsqueeze(1)).t())
        return y if s["bias"] is None else y.add_(d["bias"])
    if s["op"] == "weight_grad":
        kept = _kept64(d["x"])
        if s["rstd"] is not None:
            kept = kept * d["rstd"].unsqueeze(1) * d["w"].unsqueeze(0)
        return torch.mm(d["dy"].t(), kept)
    h = d["x"] + d["residual"]
    r = 1 / torch.sqrt(torch.mean(h ** 2, 1, True) + EPS)
    y = h * r * d["w"]
    if s["op"] == "norm_q8":
        step = torch.max(torch.abs(y), 1, True).values / 127
        return {"n": step * torch.round(y / torch.where(step > 0, step, torch.ones_like(step))), "h": h}
    z = _kept64(h) * r
    dz = d["dn"] * d["w"]
    dx = d["dh"] + r * dz - r * z * torch.sum(dz * z, 1, True) / h.shape[1]
    return {"n": y, "h": h, "dx": dx, "dw": torch.einsum("mk,mk->k", d["dn"], z)}
