"""The dense operators around the routed experts, as cases that can be timed and compared.

Three operators, each as plain torch operations in 32 bits and as the framework's own call:

* ``linear``: y = x W^T with MXFP4 weights in the checkpoint layout (E2M1 pairs, low nibble = even k, and one UE8M0 scale
  per 32 k) and BF16 activations, or E4M3 activations with UE8M0 K32 scales; one token to a prefill batch.
* ``gated``: silu(x Wg^T) * (x Wu^T) with both projections in that format.
* ``norm``: the step between two blocks: the block's output (up to eight rank planes summed in rank order), its RMS norm,
  gate and scale, the residual, and the RMS norm in front of the next block.

``own = False`` computes the plain forms; ``own = True`` calls ``mimo26f_afd_b200``.
"""
import math

import torch

own = False

HIDDEN, INTER = 4096, 2048          # the layer's hidden width and an expert's intermediate width
MAX_MACS = 2 * 8192 * INTER * HIDDEN
MAX_ELEMS = 8192 * HIDDEN
EPS = 1e-6
E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def listed():
    return [
        # one token through the down projection of an expert-sized dense block: the smallest call, all latency
        {"name": "linear 1 token", "op": "linear", "rows": 1, "n": HIDDEN, "k": INTER, "x": "bf16", "out": "bf16", "pad": 0},
        # one token through the down projection of a dense block four times as wide as the hidden state
        {"name": "linear 1 token wide", "op": "linear", "rows": 1, "n": HIDDEN, "k": 4 * HIDDEN, "x": "bf16", "out": "bf16", "pad": 0},
        # the 16-token decode batch; FP32 out, as a tensor-parallel rank's partial sum is kept
        {"name": "linear 16 tokens", "op": "linear", "rows": 16, "n": HIDDEN, "k": 4 * HIDDEN, "x": "bf16", "out": "f32", "pad": 0},
        # a ragged batch, an odd output width, k no multiple of 128, padded rows, activations that arrive quantised
        {"name": "linear 77 tokens ragged", "op": "linear", "rows": 77, "n": 1001, "k": 4064, "x": "e4m3", "out": "bf16", "pad": 32},
        # a chunk of prefill on quantised rows
        {"name": "linear 2048 tokens e4m3", "op": "linear", "rows": 2048, "n": HIDDEN, "k": HIDDEN, "x": "e4m3", "out": "bf16", "pad": 0},
        # the 8,192-token prefill batch through the down projection
        {"name": "linear 8192 tokens", "op": "linear", "rows": 8192, "n": HIDDEN, "k": INTER, "x": "bf16", "out": "bf16", "pad": 0},
        # one token through gate and up of an expert-sized dense block
        {"name": "gated 1 token", "op": "gated", "rows": 1, "n": INTER, "k": HIDDEN, "x": "bf16", "out": "bf16", "pad": 0},
        # the 16-token decode batch through gate and up of the wide dense block
        {"name": "gated 16 tokens wide", "op": "gated", "rows": 16, "n": 4 * HIDDEN, "k": HIDDEN, "x": "bf16", "out": "bf16", "pad": 0},
        # the 8,192-token prefill batch through gate and up
        {"name": "gated 8192 tokens", "op": "gated", "rows": 8192, "n": INTER, "k": HIDDEN, "x": "bf16", "out": "bf16", "pad": 0},
        # one token between two blocks
        {"name": "norm 1 token", "op": "norm", "rows": 1, "width": HIDDEN, "planes": 1, "y": "bf16", "h": "f32", "n": "bf16", "post": True, "gate": "channel", "pad": 0},
        # four ranks' planes of a ragged batch, an odd width, a gate per token (a shared expert's), FP32 out
        {"name": "norm 333 tokens ragged", "op": "norm", "rows": 333, "width": HIDDEN - 1, "planes": 4, "y": "bf16", "h": "f32", "n": "f32", "post": True, "gate": "token", "pad": 5},
        # prefill, BF16 residual stream, a gate per element
        {"name": "norm 8192 tokens", "op": "norm", "rows": 8192, "width": HIDDEN, "planes": 1, "y": "bf16", "h": "bf16", "n": "bf16", "post": True, "gate": "element", "pad": 0},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("linear", "linear", "gated", "gated", "norm", "norm"))
    if op == "norm":
        width = _log(rng, 64, 4 * HIDDEN)
        if rng.random() < 0.5:
            width = max(8, width // 8 * 8)
        rows = min(_log(rng, 1, 8192), max(1, MAX_ELEMS // (2 * width)))
        y = rng.choice(("bf16", "bf16", "f32"))
        return {"op": op, "rows": rows, "width": width, "planes": rng.choice((1, 1, 2, 4, 8)) if y == "bf16" else 1, "y": y,
                "h": rng.choice(("f32", "bf16")), "n": rng.choice(("bf16", "f32")), "post": rng.random() < 0.7,
                "gate": rng.choice(("none", "token", "channel", "element")), "pad": rng.choice((0, 0, 3, 8))}
    n = _log(rng, 64, 4 * HIDDEN)
    if rng.random() < 0.5:
        n = max(64, n // 64 * 64)
    k = 32 * _log(rng, 4, 4 * HIDDEN // 32)
    macs = MAX_MACS // (2 if op == "gated" else 1)
    rows = max(1, min(_log(rng, 1, 8192), macs // (n * k)))
    x = rng.choice(("bf16", "bf16", "e4m3"))
    return {"op": op, "rows": rows, "n": n, "k": k, "x": x, "out": rng.choice(("bf16", "f32")), "pad": rng.choice((0, 0, 16, 40))}


# ------------------------------------------------------------------------------------------------------------- inputs
TYPES = {"bf16": torch.bfloat16, "f32": torch.float32}


def _weights(n, k, gen):
    """MXFP4 in the checkpoint layout: all sixteen codes, scale bytes 118..122 as in the synthetic layers."""
    w = torch.randint(0, 256, (n, k // 2), dtype=torch.uint8, device="cuda", generator=gen)
    s = torch.randint(118, 123, (n, k // 32), dtype=torch.uint8, device="cuda", generator=gen)
    return w, s


def _activations(rows, k, gen):
    """Normal values with a few channels far above the rest, as a residual stream has them."""
    x = torch.randn(rows, k, device="cuda", generator=gen)
    loud = torch.rand(k, device="cuda", generator=gen) < 0.004
    return (x * torch.where(loud, 30.0, 1.0)).to(torch.bfloat16)


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    rows, st = case["rows"], dict(case)
    if case["op"] == "norm":
        width, pitch = case["width"], case["width"] + case["pad"]
        yt, ht = TYPES[case["y"]], TYPES[case["h"]]

        def rows_of(t):
            return torch.randn(rows, pitch, device="cuda", generator=gen).to(t)[:, :width]

        st["planes"] = [rows_of(yt) for _ in range(case["planes"])]
        st["residual"] = (4.0 * torch.randn(rows, pitch, device="cuda", generator=gen)).to(ht)[:, :width]
        st["pre_w"] = 1.0 + 0.1 * torch.randn(width, device="cuda", generator=gen)
        st["post_w"] = 1.0 + 0.1 * torch.randn(width, device="cuda", generator=gen) if case["post"] else None
        st["gate"] = None
        if case["gate"] == "token":
            st["gate"] = torch.rand(rows, device="cuda", generator=gen)
        elif case["gate"] == "channel":
            st["gate"] = torch.rand(width, device="cuda", generator=gen)
        elif case["gate"] == "element":
            st["gate"] = rows_of(yt)
        st["gate_kind"] = case["gate"]
        st["h_out"] = torch.empty(rows, pitch, dtype=ht, device="cuda")[:, :width]
        st["n_out"] = torch.empty(rows, pitch, dtype=TYPES[case["n"]], device="cuda")[:, :width]
        return st
    n, k, pad = case["n"], case["k"], case["pad"]
    x = torch.zeros(rows, k + pad, dtype=torch.bfloat16, device="cuda")
    x[:, :k] = _activations(rows, k, gen)
    if case["x"] == "e4m3":
        v = x[:, :k].float().view(rows, k // 32, 32)
        e = torch.ceil(torch.log2(v.abs().amax(-1).clamp_min(2.0**-100) / 448.0))
        q = torch.zeros(rows, k + pad, dtype=torch.uint8, device="cuda")
        q[:, :k] = (v * torch.exp2(-e)[..., None]).clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8).view(rows, k)
        st["x_values"], st["x_scales"] = q[:, :k], (e + 127).to(torch.uint8)
    else:
        st["x_values"], st["x_scales"] = x[:, :k], None
    st["w"] = [_weights(n, k, gen) for _ in range(2 if case["op"] == "gated" else 1)]
    st["y"] = torch.empty(rows, n + pad, dtype=TYPES[case["out"]], device="cuda")[:, :n]
    if own:
        import mimo26f_afd_b200 as M

        flat = [t for pair in st["w"] for t in pair]
        st["layer"] = (M.Linear.gated if case["op"] == "gated" else M.Linear.new)(*flat, n, k)
        st["workspace"] = torch.empty(max(1, st["layer"].workspace_bytes(rows)), dtype=torch.uint8, device="cuda")
        st["fault"] = torch.zeros(1, dtype=torch.int32, device="cuda")
    return st


# --------------------------------------------------------------------------------------------------------- plain forms
def _weight_f32(w, s):
    table = torch.tensor(E2M1 + tuple(-v for v in E2M1), device=w.device)
    codes = torch.stack((w & 15, w >> 4), dim=-1).flatten(1)
    return table[codes.int()] * torch.exp2(s.float() - 127.0).repeat_interleave(32, dim=1)


def _x_f32(st):
    if st["x_scales"] is None:
        return st["x_values"].float()
    return st["x_values"].contiguous().view(torch.float8_e4m3fn).float() * torch.exp2(st["x_scales"].float() - 127.0).repeat_interleave(32, dim=1)


def _plain_product(st):
    x = _x_f32(st)
    y = x @ _weight_f32(*st["w"][0]).t()
    if st["op"] == "gated":
        y = y / (1.0 + torch.exp(-y)) * (x @ _weight_f32(*st["w"][1]).t())
    return y.to(TYPES[st["out"]])


def _plain_norm(st):
    y = sum(p.float() for p in st["planes"])
    if st["post_w"] is not None:
        y = y * torch.rsqrt((y * y).mean(-1, keepdim=True) + EPS) * st["post_w"]
    if st["gate"] is not None:
        y = y * (st["gate"][:, None] if st["gate_kind"] == "token" else st["gate"].float())
    h = 0.5 * st["residual"].float() + 1.25 * y
    n = h * torch.rsqrt((h * h).mean(-1, keepdim=True) + EPS) * st["pre_w"]
    return {"h": h.to(st["h_out"].dtype), "n": n.to(st["n_out"].dtype)}


def run(state):
    st = state
    if not own:
        return _plain_norm(st) if st["op"] == "norm" else _plain_product(st)
    import mimo26f_afd_b200 as M

    stream = torch.cuda.current_stream().cuda_stream
    if st["op"] == "norm":
        kinds = {"none": M.GATE_NONE, "token": M.GATE_TOKEN, "channel": M.GATE_CHANNEL, "element": M.GATE_ELEMENT}
        M.block_norm_dev(st["planes"], st["residual"], st["rows"], st["width"], post_w=st["post_w"], gate=st["gate"],
                         gate_kind=kinds[st["gate_kind"]], y_dtype=0 if st["y"] == "bf16" else 1, y_pitch=st["width"] + st["pad"],
                         y_scale=1.25, h_dtype=0 if st["h"] == "bf16" else 1, h_pitch=st["width"] + st["pad"], residual_scale=0.5,
                         pre_w=st["pre_w"], w_dtype=1, eps=EPS, h_out=st["h_out"], n_out=st["n_out"],
                         n_dtype=0 if st["n"] == "bf16" else 1, n_pitch=st["width"] + st["pad"], stream=stream)
        return {"h": st["h_out"], "n": st["n_out"]}
    M.linear_dev(st["layer"], st["x_values"], st["rows"], st["y"], x_dtype=2 if st["x"] == "e4m3" else 0, x_scales=st["x_scales"],
                 x_pitch=st["k"] + st["pad"], y_dtype=0 if st["out"] == "bf16" else 1, y_pitch=st["n"] + st["pad"],
                 workspace=st["workspace"], fault=st["fault"], stream=stream)
    return st["y"]


def work(case):
    rows = case["rows"]
    size = {"bf16": 2, "f32": 4}
    if case["op"] == "norm":
        width = case["width"]
        gate = {"none": 0, "token": 4 * rows, "channel": 4 * width, "element": rows * width * size[case["y"]]}[case["gate"]]
        per = case["planes"] * size[case["y"]] + 2 * size[case["h"]] + size[case["n"]]
        return {"bytes": rows * width * per + gate + 4 * width * (2 if case["post"] else 1), "flops": rows * width * (case["planes"] + 12)}
    n, k = case["n"], case["k"]
    mats = 2 if case["op"] == "gated" else 1
    x = rows * k * 2 if case["x"] == "bf16" else rows * (k + k // 32)
    return {"bytes": mats * (n * k // 2 + n * k // 32) + x + rows * n * size[case["out"]], "flops": 2 * mats * rows * n * k}


# --------------------------------------------------------------------------------------------------------- in 64 bits
def _e2m1_f64(code):
    e, m = (code >> 1) & 3, code & 1
    mag = torch.where(e == 0, 0.5 * m, torch.ldexp(1.0 + 0.5 * m.double(), e.double() - 1.0))
    return torch.where(code >= 8, -mag, mag)


def _e4m3_f64(code):
    c = code.to(torch.int32)
    e, m = (c >> 3) & 15, (c & 7).double()
    mag = torch.where(e == 0, m * 2.0**-9, (1.0 + m / 8.0) * torch.pow(2.0, e.double() - 7.0))
    return torch.where(c >= 128, -mag, mag)


def _matrix_f64(w, s):
    out = torch.empty(w.shape[0], 2 * w.shape[1], dtype=torch.float64, device=w.device)
    c = w.to(torch.int32)
    out[:, 0::2] = _e2m1_f64(c & 15)
    out[:, 1::2] = _e2m1_f64(c >> 4)
    scale = torch.pow(torch.tensor(2.0, dtype=torch.float64, device=w.device), s.double() - 127.0)
    return (out.view(w.shape[0], -1, 32) * scale[:, :, None]).flatten(1)


def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "norm":
        y = torch.zeros(case["rows"], case["width"], dtype=torch.float64, device="cuda")
        for p in st["planes"]:
            y += p.double()
        if st["post_w"] is not None:
            y = y / (y.square().sum(-1, keepdim=True) / case["width"] + EPS).sqrt() * st["post_w"].double()
        if case["gate"] == "token":
            y = y * st["gate"].double().unsqueeze(1)
        elif case["gate"] != "none":
            y = y * st["gate"].double()
        h = st["residual"].double() / 2 + y * 1.25
        return {"h": h, "n": h / (h.square().sum(-1, keepdim=True) / case["width"] + EPS).sqrt() * st["pre_w"].double()}
    if case["x"] == "e4m3":
        x = _e4m3_f64(st["x_values"]).view(case["rows"], -1, 32)
        x = (x * torch.pow(2.0, st["x_scales"].double() - 127.0)[:, :, None]).flatten(1)
    else:
        x = st["x_values"].double()
    y = torch.mm(x, _matrix_f64(*st["w"][0]).T)
    if case["op"] == "gated":
        y = y * torch.sigmoid(y) * torch.mm(x, _matrix_f64(*st["w"][1]).T)
    return y
