"""The dense operators on a B200 against their formulas in 64 bits.

Bounds, per output, from the arithmetic alone (u = 2^-24, the FP32 half step; S = sum |x w| over k):
* product: a K32 block of BF16 activations is exact save for elements below 2^-13 of its largest, off by at most 2^-21 of that
  largest (times sum |w| of the block); the tensor core adds the block products and the FP32 running sum with at most one
  truncation (2 u) each: two pieces x k / 32 blocks, 32 products in each, up to eight partial sums: (k / 16 + 48) 2 u S.
* gated: |silu'| <= 1.1, so 1.1 |u| dg + |silu(g)| du, plus 2^-19 |y| for the activation's own arithmetic.
* norm: at most 8 planes and a reduction tree: 64 u relative on every factor.
* one rounding to BF16: 2^-8 |y| (half a step is eps / 2 = 2^-8 relative).
"""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

U = 2.0**-24


@pytest.fixture(scope="module")
def torch():
    import torch

    assert torch.cuda.is_available(), "these tests need the GPU box"
    return torch


def gen(torch, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def make_weights(torch, n, k, g, lo=118, hi=122):
    w = torch.randint(0, 256, (n, k // 2), dtype=torch.uint8, device="cuda", generator=g)
    s = torch.randint(lo, hi + 1, (n, k // 32), dtype=torch.uint8, device="cuda", generator=g)
    return w, s


def weight_f64(torch, w, s):
    mags = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64, device="cuda")
    table = torch.cat((mags, -mags))
    codes = torch.stack((w & 15, w >> 4), -1).flatten(1).long()
    sc = torch.exp2(torch.where(s == 255, 254, s.int()).double() - 127)
    return table[codes] * sc.repeat_interleave(32, 1)


def e4m3_f64(torch, q, xs):
    return q.contiguous().view(torch.float8_e4m3fn).double() * torch.exp2(xs.double() - 127).repeat_interleave(32, 1)


def product_and_bound(torch, x, W, quantised=False):
    """y and its bound in 64 bits; x [rows, k], W [n, k]."""
    k = x.shape[1]
    y = x @ W.T
    bound = (k / 16 + 48) * 2 * U * (x.abs() @ W.abs().T)
    if not quantised:
        amax = x.abs().view(x.shape[0], -1, 32).amax(-1)
        bound = bound + 2.0**-21 * (amax @ W.abs().view(W.shape[0], -1, 32).sum(-1).T)
    return y, bound


def rounded(y, bound, bf16):
    return bound + (2.0**-8 * (y.abs() + bound) if bf16 else U * y.abs())


class Runner:
    def __init__(self, torch, layer, rows):
        self.torch, self.layer = torch, layer
        self.ws = torch.empty(layer.workspace_bytes(rows), dtype=torch.uint8, device="cuda")
        self.fault = torch.zeros(1, dtype=torch.int32, device="cuda")

    def __call__(self, x, rows, *, f32=True, x_scales=None, x_pitch=0, y=None, y_pitch=0, stream=None):
        import mimo26f_afd_b200 as M

        torch = self.torch
        if y is None:
            y = torch.empty(rows, self.layer.n, dtype=torch.float32 if f32 else torch.bfloat16, device="cuda")
        M.linear_dev(self.layer, x, rows, y, x_dtype=0 if x_scales is None else 2, x_scales=x_scales, x_pitch=x_pitch, y_dtype=int(f32), y_pitch=y_pitch,
                     workspace=self.ws, fault=self.fault, stream=stream)
        return y


def check(torch, got, want, bound):
    torch.cuda.synchronize()
    off = (got.double() - want).abs()
    worst = float((off / bound.clamp_min(1e-300)).max())
    assert bool((off <= bound).all()), f"worst error {worst:.3g} of its bound"


# ------------------------------------------------------------------------------------------------------------- linear
@pytest.mark.parametrize("rows", [1, 2, 7, 15, 16, 17, 31, 32, 33, 64, 65, 100, 128, 129, 200, 256, 257, 700])
@pytest.mark.parametrize("n,k", [(256, 512), (130, 160)])
def test_linear_rows(torch, rows, n, k):
    import mimo26f_afd_b200 as M

    g = gen(torch, rows * 7 + n)
    w, s = make_weights(torch, n, k, g)
    x = (torch.randn(rows, k, device="cuda", generator=g) * torch.exp2(torch.randint(-8, 8, (rows, k // 32), device="cuda", generator=g).float()).repeat_interleave(32, 1)).to(torch.bfloat16)
    run = Runner(torch, M.Linear.new(w, s, n, k), rows)
    y, bound = product_and_bound(torch, x.double(), weight_f64(torch, w, s))
    check(torch, run(x, rows), y, rounded(y, bound, False))
    check(torch, run(x, rows, f32=False), y, rounded(y, bound, True))
    assert int(run.fault) == 0


@pytest.mark.parametrize("n", [1, 2, 63, 64, 65, 127, 128, 129, 1000, 4096])
@pytest.mark.parametrize("k", [32, 64, 128, 416, 4096])
def test_linear_extents(torch, n, k):
    import mimo26f_afd_b200 as M

    g = gen(torch, n * 31 + k)
    w, s = make_weights(torch, n, k, g)
    rows = 5
    x = torch.randn(rows, k, device="cuda", generator=g).to(torch.bfloat16)
    run = Runner(torch, M.Linear.new(w, s, n, k), rows)
    y, bound = product_and_bound(torch, x.double(), weight_f64(torch, w, s))
    check(torch, run(x, rows), y, rounded(y, bound, False))


@pytest.mark.parametrize("rows", [1, 3, 8, 13, 16, 23, 32, 41, 64, 90, 120, 127, 128])
@pytest.mark.parametrize("n", [9000, 30000])
def test_many_weight_tiles_with_many_chunks_each(torch, rows, n):
    """Enough tiles that K is hardly split: every stage of the pipeline is reused several times in one CTA."""
    import mimo26f_afd_b200 as M

    k = 4096
    g = gen(torch, rows + n)
    w, s = make_weights(torch, n, k, g)
    x = torch.randn(rows, k, device="cuda", generator=g).to(torch.bfloat16)
    q = torch.randint(0, 127, (rows, k), dtype=torch.uint8, device="cuda", generator=g)
    xs = torch.randint(110, 130, (rows, k // 32), dtype=torch.uint8, device="cuda", generator=g)
    run = Runner(torch, M.Linear.new(w, s, n, k), rows)
    W = weight_f64(torch, w, s)
    y, bound = product_and_bound(torch, x.double(), W)
    check(torch, run(x, rows), y, rounded(y, bound, False))
    y, bound = product_and_bound(torch, e4m3_f64(torch, q, xs), W, quantised=True)
    check(torch, run(q, rows, x_scales=xs), y, rounded(y, bound, False))
    assert int(run.fault) == 0


@pytest.mark.parametrize("rows", [1, 16, 40, 130])
@pytest.mark.parametrize("n,k", [(64, 128), (65, 160), (320, 4096), (1, 32), (129, 96), (200, 1024)])
def test_gated(torch, rows, n, k):
    import mimo26f_afd_b200 as M

    g = gen(torch, rows + n + k)
    gw, gs = make_weights(torch, n, k, g)
    uw, us = make_weights(torch, n, k, g)
    x = torch.randn(rows, k, device="cuda", generator=g).to(torch.bfloat16)
    run = Runner(torch, M.Linear.gated(gw, gs, uw, us, n, k), rows)
    a, da = product_and_bound(torch, x.double(), weight_f64(torch, gw, gs))
    b, db = product_and_bound(torch, x.double(), weight_f64(torch, uw, us))
    silu = a * torch.sigmoid(a)
    y = silu * b
    bound = 1.1 * da * (b.abs() + db) + silu.abs() * db + 2.0**-19 * y.abs()
    check(torch, run(x, rows), y, rounded(y, bound, False))
    check(torch, run(x, rows, f32=False), y, rounded(y, bound, True))
    assert int(run.fault) == 0


@pytest.mark.parametrize("rows", [1, 16, 33, 130, 300])
@pytest.mark.parametrize("gated", [False, True])
def test_quantised_activations(torch, rows, gated):
    import mimo26f_afd_b200 as M

    n, k = 200, 416
    g = gen(torch, rows)
    ws = [make_weights(torch, n, k, g) for _ in range(1 + gated)]
    q = torch.randint(0, 256, (rows, k), dtype=torch.uint8, device="cuda", generator=g)
    q[(q & 127) == 127] = 0x38                                  # no NaN codes
    xs = torch.randint(110, 130, (rows, k // 32), dtype=torch.uint8, device="cuda", generator=g)
    layer = M.Linear.gated(*ws[0], *ws[1], n, k) if gated else M.Linear.new(*ws[0], n, k)
    run = Runner(torch, layer, rows)
    x = e4m3_f64(torch, q, xs) * (2.0**-9 if gated else 1.0)    # gated: keep the activation's argument moderate
    if gated:
        xs = xs - 9
    y, bound = product_and_bound(torch, x, weight_f64(torch, *ws[0]), quantised=True)
    if gated:
        b, db = product_and_bound(torch, x, weight_f64(torch, *ws[1]), quantised=True)
        silu = y * torch.sigmoid(y)
        bound = 1.1 * bound * (b.abs() + db) + silu.abs() * db + 2.0**-19 * (silu * b).abs()
        y = silu * b
    check(torch, run(q, rows, x_scales=xs), y, rounded(y, bound, False))


@pytest.mark.parametrize("rows", [129, 136, 150, 256, 257, 273, 384, 385, 400, 511, 512, 700])
@pytest.mark.parametrize("k", [32, 160, 1152])
def test_enough_work_for_cta_pairs(torch, rows, k):
    """At least a quarter as many 256-row x 256-token items as SMs: linear and gated, both kinds of activations, both output types."""
    import mimo26f_afd_b200 as M

    g = gen(torch, rows + k)
    n = 9601
    w, s = make_weights(torch, n, k, g)
    x = torch.randn(rows, k, device="cuda", generator=g).to(torch.bfloat16)
    q = torch.randint(0, 127, (rows, k), dtype=torch.uint8, device="cuda", generator=g)
    xs = torch.randint(112, 118, (rows, k // 32), dtype=torch.uint8, device="cuda", generator=g)
    W = weight_f64(torch, w, s)
    run = Runner(torch, M.Linear.new(w, s, n, k), rows)
    y, bound = product_and_bound(torch, x.double(), W)
    check(torch, run(x, rows), y, rounded(y, bound, False))
    yq, bq = product_and_bound(torch, e4m3_f64(torch, q, xs), W, quantised=True)
    check(torch, run(q, rows, x_scales=xs, f32=False), yq, rounded(yq, bq, True))
    half = n // 2
    gated = Runner(torch, M.Linear.gated(w[:half].contiguous(), s[:half].contiguous(), w[half:2 * half].contiguous(), s[half:2 * half].contiguous(), half, k), rows)
    for a, da, got in ((y, bound, gated(x, rows, f32=False)), (yq, bq, gated(q, rows, x_scales=xs, f32=False))):
        b, db, a, da = a[:, half:2 * half], da[:, half:2 * half], a[:, :half], da[:, :half]
        silu = a * torch.sigmoid(a)
        check(torch, got, silu * b, rounded(silu * b, 1.1 * da * (b.abs() + db) + silu.abs() * db + 2.0**-19 * (silu * b).abs(), True))
    assert int(run.fault) == 0 and int(gated.fault) == 0


@pytest.mark.parametrize("rows", [129, 135, 200, 256, 300, 520, 1000])
@pytest.mark.parametrize("n,k", [(60, 96), (500, 1024), (130, 2048)])
def test_several_token_tiles_converted_in_the_kernel(torch, rows, n, k):
    import mimo26f_afd_b200 as M

    g = gen(torch, rows + n)
    w, s = make_weights(torch, n, k, g)
    W = weight_f64(torch, w, s)
    x = torch.randn(rows, k, device="cuda", generator=g).to(torch.bfloat16)
    q = torch.randint(0, 127, (rows, k), dtype=torch.uint8, device="cuda", generator=g)
    xs = torch.randint(110, 130, (rows, k // 32), dtype=torch.uint8, device="cuda", generator=g)
    run = Runner(torch, M.Linear.new(w, s, n, k), rows)
    y, bound = product_and_bound(torch, x.double(), W)
    check(torch, run(x, rows), y, rounded(y, bound, False))
    y, bound = product_and_bound(torch, e4m3_f64(torch, q, xs), W, quantised=True)
    check(torch, run(q, rows, x_scales=xs), y, rounded(y, bound, False))
    assert int(run.fault) == 0


def test_cta_pairs_with_many_items_each(torch):
    import mimo26f_afd_b200 as M

    n, k, rows = 4096, 2048, 4000
    g = gen(torch, 77)
    w, s = make_weights(torch, n, k, g)
    x = torch.randn(rows, k, device="cuda", generator=g).to(torch.bfloat16)
    run = Runner(torch, M.Linear.new(w, s, n, k), rows)
    y, bound = product_and_bound(torch, x.double(), weight_f64(torch, w, s))
    a = run(x, rows).clone()
    check(torch, a, y, rounded(y, bound, False))
    x2 = x.clone()
    x2[1::2] = x[0::2]
    b = run(x2, rows)
    torch.cuda.synchronize()
    assert torch.equal(a[0::2], b[0::2]) and int(run.fault) == 0


def test_bf16_activations_pass_unquantised(torch):
    """One weight of 1.0 per row: the output is the activation itself, bit for bit down to 2^-13.8 of its block's largest (2^-6 / 224 at
    the worst: the block's scale leaves its largest in 224..448)."""
    import mimo26f_afd_b200 as M

    k = 256
    w = torch.zeros(k, k // 2, dtype=torch.uint8, device="cuda")
    i = torch.arange(k, device="cuda")
    w[i, i // 2] = torch.where(i % 2 == 0, 0x02, 0x20).to(torch.uint8)
    s = torch.full((k, k // 32), 127, dtype=torch.uint8, device="cuda")
    rows = 64
    g = gen(torch, 5)
    x = torch.randn(rows, k, device="cuda", generator=g) * torch.exp2(torch.randint(-30, 1, (rows, k), device="cuda", generator=g).float())
    x = (x * torch.exp2(torch.randint(-60, 60, (rows, 1), device="cuda", generator=g).float())).to(torch.bfloat16)
    x[0] = 0.0
    y = Runner(torch, M.Linear.new(w, s, k, k), rows)(x, rows)
    torch.cuda.synchronize()
    amax = x.abs().float().view(rows, -1, 32).amax(-1).repeat_interleave(32, 1)
    large = x.abs().float() >= amax * 2.0**-13.8
    assert 0.3 < float(large.float().mean()) < 0.8
    assert torch.equal(y[large], x.float()[large])
    assert bool(((y - x.float()).abs() <= amax * 2.0**-21).all())


@pytest.mark.parametrize("bad", [float("inf"), float("-inf"), float("nan")])
def test_a_row_with_a_nonfinite_value_is_nan_and_the_others_are_untouched(torch, bad):
    import mimo26f_afd_b200 as M

    n, k, rows = 192, 256, 20
    g = gen(torch, 9)
    w, s = make_weights(torch, n, k, g)
    x = torch.randn(rows, k, device="cuda", generator=g).to(torch.bfloat16)
    run = Runner(torch, M.Linear.new(w, s, n, k), rows)
    want = run(x, rows).clone()
    x[3, 77] = bad
    y = run(x, rows)
    torch.cuda.synchronize()
    assert bool(torch.isnan(y[3]).all())
    keep = torch.arange(rows, device="cuda") != 3
    assert torch.equal(y[keep], want[keep])


def test_quantised_rows_with_nan_codes_or_scales_are_nan(torch):
    import mimo26f_afd_b200 as M

    n, k = 9728, 128
    g = gen(torch, 10)
    w, s = make_weights(torch, n, k, g)
    layer = M.Linear.new(w, s, n, k)
    for rows in (6, 70, 500):                                   # converted in the kernel, staged, on CTA pairs
        for pitch in (k, k + 8):                                # rows TMA can take in place, and not
            q = torch.full((rows, pitch), 0x38, dtype=torch.uint8, device="cuda")[:, :k]
            xs = torch.full((rows, k // 32), 127, dtype=torch.uint8, device="cuda")
            q[1, 40] = 0x7f
            q[2, 127] = 0xff
            xs[4, 3] = 255
            y = Runner(torch, layer, rows)(q, rows, x_scales=xs, x_pitch=pitch)
            torch.cuda.synchronize()
            nan = torch.isnan(y)
            want = [i in (1, 2, 4) for i in range(rows)]
            assert nan.all(1).tolist() == want and nan.any(1).tolist() == want


def test_scale_bytes_at_the_ends_of_their_range(torch):
    """Weight scales 0..254 and 255 (stored as 254): one byte per row, activations that keep the product inside FP32."""
    import mimo26f_afd_b200 as M

    n, k, rows = 256, 32, 4
    w = torch.full((n, k // 2), 0x22, dtype=torch.uint8, device="cuda")
    w[:, 0] = 0x02                                              # 31 weights of 1.0
    s = torch.arange(256, device="cuda").to(torch.uint8).view(n, 1)
    g = gen(torch, 11)
    for shift, keep in ((-20.0, slice(60, 256)), (20.0, slice(0, 200))):
        x = (torch.randn(rows, k, device="cuda", generator=g) * 2.0**shift).to(torch.bfloat16)
        y, bound = product_and_bound(torch, x.double(), weight_f64(torch, w, s))
        got = Runner(torch, M.Linear.new(w, s, n, k), rows)(x, rows)
        torch.cuda.synchronize()
        off = (got.double() - y).abs()[:, keep]
        assert bool((off <= (rounded(y, bound, False) + 2.0**-126)[:, keep]).all())


@pytest.mark.parametrize("rows", [3, 20, 40, 150])
@pytest.mark.parametrize("x_off,x_pad,y_off,y_pad", [(0, 8, 0, 5), (1, 3, 1, 0), (3, 0, 2, 7), (8, 16, 0, 64)])
def test_pitches_and_alignment_and_what_lies_between_the_rows(torch, rows, x_off, x_pad, y_off, y_pad):
    import mimo26f_afd_b200 as M

    n, k = 130, 224
    g = gen(torch, rows + x_off)
    w, s = make_weights(torch, n, k, g)
    xb = torch.full((x_off + rows * (k + x_pad),), float("nan"), dtype=torch.bfloat16, device="cuda")
    x = torch.as_strided(xb, (rows, k), (k + x_pad, 1), x_off)
    x.copy_(torch.randn(rows, k, device="cuda", generator=g))
    layer = M.Linear.new(w, s, n, k)
    run = Runner(torch, layer, rows)
    y, bound = product_and_bound(torch, x.double(), weight_f64(torch, w, s))
    for f32 in (True, False):
        dt = torch.float32 if f32 else torch.bfloat16
        yb = torch.full((y_off + (rows + 1) * (n + y_pad),), -77.0, dtype=dt, device="cuda")
        yv = torch.as_strided(yb, (rows, n), (n + y_pad, 1), y_off)
        run(x, rows, f32=f32, x_pitch=k + x_pad, y=yv, y_pitch=n + y_pad)
        check(torch, yv, y, rounded(y, bound, not f32))
        yv.fill_(-77.0)
        assert bool((yb == -77.0).all())                        # nothing outside the rows was written


@pytest.mark.parametrize("rows", [3, 40, 150])
@pytest.mark.parametrize("off,pad", [(0, 0), (0, 16), (0, 8), (1, 0), (4, 4), (8, 3), (16, 32)])
def test_quantised_rows_of_any_alignment(torch, rows, off, pad):
    import mimo26f_afd_b200 as M

    n, k = 70, 160
    g = gen(torch, rows + off)
    w, s = make_weights(torch, n, k, g)
    qb = torch.full((off + rows * (k + pad),), 0x7f, dtype=torch.uint8, device="cuda")
    q = torch.as_strided(qb, (rows, k), (k + pad, 1), off)
    q.copy_(torch.randint(0, 127, (rows, k), dtype=torch.uint8, device="cuda", generator=g))
    xs = torch.randint(110, 130, (rows, k // 32), dtype=torch.uint8, device="cuda", generator=g)
    y, bound = product_and_bound(torch, e4m3_f64(torch, q, xs), weight_f64(torch, w, s), quantised=True)
    check(torch, Runner(torch, M.Linear.new(w, s, n, k), rows)(q, rows, x_scales=xs, x_pitch=k + pad), y, rounded(y, bound, False))


def test_rows_more_than_four_gigabytes_apart(torch):
    """Offsets past 32 bits, in bytes and in elements."""
    import mimo26f_afd_b200 as M

    n, k, pitch = 64, 64, (1 << 32) + 64
    g = gen(torch, 17)
    w, s = make_weights(torch, n, k, g)
    xb, yb = (torch.empty(pitch + 64, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    x, y = (torch.as_strided(b, (2, 64), (pitch, 1)) for b in (xb, yb))
    x.copy_(torch.randn(2, k, device="cuda", generator=g))
    want, bound = product_and_bound(torch, x.double(), weight_f64(torch, w, s))
    run = Runner(torch, M.Linear.new(w, s, n, k), 2)
    check(torch, run(x, 2, x_pitch=pitch, y=y, y_pitch=pitch, f32=False), want, rounded(want, bound, True))
    for width in (64, 63, 61):                                    # rows in vectors of eight, of four, and element by element
        off = 1 if width == 61 else 0
        xv, out = (torch.as_strided(b, (2, width), (pitch, 1), off) for b in (xb, yb))
        out.zero_()
        M.block_norm_dev([xv], None, 2, width, y_pitch=pitch, n_out=out, n_pitch=pitch)
        torch.cuda.synchronize()
        _, want = norm_f64([xv], None, None, None, 0, None, 1e-6, 1.0, 1.0)
        assert bool(((out.double() - want).abs() <= (2.0**-8 + 64 * U) * want.abs()).all())


def test_first_calls_inside_a_capture(torch):
    """A fresh process whose first call of every variant is captured (nothing may need a call outside before), then replayed."""
    import subprocess
    import sys

    from conftest import ROOT

    code = """
import sys; sys.path.insert(0, %r)
import torch, mimo26f_afd_b200 as M
def mk(n, k):
    return torch.randint(0, 256, (n, k // 2), dtype=torch.uint8, device='cuda'), torch.full((n, k // 32), 120, dtype=torch.uint8, device='cuda')
n, k = 9600, 256
w, s = mk(n, k)
lin, gat = M.Linear.new(w, s, n, k), M.Linear.gated(w, s, w, s, n, k)
fault = torch.zeros(1, dtype=torch.int32, device='cuda')
ws = torch.empty(lin.workspace_bytes(600), dtype=torch.uint8, device='cuda')
jobs = []
for rows in (1, 20, 50, 100, 600):
    x = torch.randn(rows, k, device='cuda').bfloat16()
    jobs.append((x, torch.zeros(rows, n, device='cuda'), torch.zeros(rows, n, device='cuda'), torch.zeros(rows, k, device='cuda'), torch.zeros(rows, k - 1, device='cuda')))
torch.cuda.synchronize()
def run(st):
    for x, a, b, h, h1 in jobs:
        r = x.shape[0]
        M.linear_dev(lin, x, r, a, y_dtype=1, workspace=ws, fault=fault, stream=st)
        M.linear_dev(gat, x, r, b, y_dtype=1, workspace=ws, fault=fault, stream=st)
        M.block_norm_dev([x], None, r, k, n_out=h, n_dtype=1, stream=st)
        M.block_norm_dev([x], None, r, k - 1, n_out=h1, n_dtype=1, stream=st)
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    run(torch.cuda.current_stream().cuda_stream)
g.replay(); torch.cuda.synchronize()
got = [[t.clone() for t in j[1:]] for j in jobs]
for j in jobs:
    for t in j[1:]: t.zero_()
run(None); torch.cuda.synchronize()
assert all(torch.equal(p, q) and float(p.abs().sum()) > 0 for o, j in zip(got, jobs) for p, q in zip(o, j[1:]))
assert int(fault) == 0
print('captured')
""" % ROOT
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "captured" in r.stdout, r.stderr[-2000:]


def test_weights_of_any_alignment(torch):
    import mimo26f_afd_b200 as M

    n, k, rows = 70, 96, 4
    g = gen(torch, 12)
    wb = torch.randint(0, 256, (n * k // 2 + 3,), dtype=torch.uint8, device="cuda", generator=g)
    sb = torch.randint(118, 123, (n * k // 32 + 1,), dtype=torch.uint8, device="cuda", generator=g)
    w, s = wb[3:].view(n, k // 2), sb[1:].view(n, k // 32)
    x = torch.randn(rows, k, device="cuda", generator=g).to(torch.bfloat16)
    y, bound = product_and_bound(torch, x.double(), weight_f64(torch, w, s))
    check(torch, Runner(torch, M.Linear.new(w, s, n, k), rows)(x, rows), y, rounded(y, bound, False))


def test_rows_do_not_depend_on_each_other_and_calls_repeat_bit_for_bit(torch):
    import mimo26f_afd_b200 as M

    n, k, rows = 320, 2048, 300
    g = gen(torch, 13)
    w, s = make_weights(torch, n, k, g)
    x = torch.randn(rows, k, device="cuda", generator=g).to(torch.bfloat16)
    run = Runner(torch, M.Linear.new(w, s, n, k), rows)
    a = run(x, rows).clone()
    x2 = x.clone()
    x2[1::2] = torch.randn(rows // 2, k, device="cuda", generator=g).to(torch.bfloat16)
    b = run(x2, rows)
    torch.cuda.synchronize()
    assert torch.equal(a[0::2], b[0::2])
    c = run(x, rows)
    torch.cuda.synchronize()
    assert torch.equal(a, c)


def test_more_rows_than_a_pass(torch):
    import mimo26f_afd_b200 as M

    n, k, rows = 64, 64, 8192 + 130
    g = gen(torch, 14)
    w, s = make_weights(torch, n, k, g)
    x = torch.randn(rows, k, device="cuda", generator=g).to(torch.bfloat16)
    run = Runner(torch, M.Linear.new(w, s, n, k), rows)
    y, bound = product_and_bound(torch, x.double(), weight_f64(torch, w, s))
    check(torch, run(x, rows), y, rounded(y, bound, False))


def test_two_streams_with_their_own_workspaces_and_a_replayed_graph(torch):
    import mimo26f_afd_b200 as M

    n, k, rows = 512, 1024, 24
    g = gen(torch, 15)
    w, s = make_weights(torch, n, k, g)
    layer = M.Linear.new(w, s, n, k)
    xs = [torch.randn(rows, k, device="cuda", generator=g).to(torch.bfloat16) for _ in range(2)]
    want = [Runner(torch, layer, rows)(x, rows).clone() for x in xs]
    torch.cuda.synchronize()
    runs = [Runner(torch, layer, rows) for _ in range(2)]
    outs = [torch.empty(rows, n, device="cuda") for _ in range(2)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(20):
        for r, x, y, st in zip(runs, xs, outs, streams):
            r(x, rows, y=y, stream=st.cuda_stream)
    torch.cuda.synchronize()
    assert torch.equal(outs[0], want[0]) and torch.equal(outs[1], want[1])

    graph = torch.cuda.CUDAGraph()
    x, y = xs[0].clone(), torch.empty(rows, n, device="cuda")
    with torch.cuda.graph(graph):
        runs[0](x, rows, y=y, stream=torch.cuda.current_stream().cuda_stream)
    for i in (1, 0):
        x.copy_(xs[i])
        y.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, want[i])


def test_calls_queued_behind_a_long_kernel(torch):
    """Everything queued while the stream is busy for longer than the bound of the kernels' own waits."""
    import mimo26f_afd_b200 as M

    n, k = 4096, 512
    g = gen(torch, 18)
    w, s = make_weights(torch, n, k, g)
    layer = M.Linear.new(w, s, n, k)
    runs = {rows: (Runner(torch, layer, rows), torch.randn(rows, k, device="cuda", generator=g).to(torch.bfloat16)) for rows in (1, 40, 2000)}
    want = {rows: r(x, rows).clone() for rows, (r, x) in runs.items()}
    outs = {rows: torch.zeros(rows, n, device="cuda") for rows in runs}
    copies = {rows: torch.empty(rows, k, dtype=torch.bfloat16, device="cuda") for rows in runs}
    torch.cuda.synchronize()
    torch.cuda._sleep(1_000_000_000)                            # about half a second
    for rows, (r, x) in runs.items():
        M.block_norm_dev([x], None, rows, k, h_dtype=0, h_out=copies[rows])      # a copy of x through the norm's kernel
        r(copies[rows], rows, y=outs[rows])
    torch.cuda.synchronize()
    for rows, (r, x) in runs.items():
        assert int(r.fault) == 0 and torch.equal(copies[rows], x) and torch.equal(outs[rows], want[rows])


def test_linear_refusals(torch):
    import mimo26f_afd_b200 as M

    n, k = 64, 64
    w, s = make_weights(torch, n, k, gen(torch, 16))
    layer = M.Linear.new(w, s, n, k)
    x = torch.zeros(40, k, dtype=torch.bfloat16, device="cuda")
    y = torch.zeros(40, n, device="cuda")
    ws = torch.empty(layer.workspace_bytes(40), dtype=torch.uint8, device="cuda")
    f = torch.zeros(1, dtype=torch.int32, device="cuda")
    ok = dict(y_dtype=1, workspace=ws, fault=f)
    M.linear_dev(layer, x, 40, y, **ok)
    M.linear_dev(layer, None, 0, None)                          # no rows: no work, nothing needed
    for rows, kw in ((4, dict(ok, x_dtype=1)), (4, dict(ok, x_dtype=3)), (4, dict(ok, y_dtype=2)), (4, dict(ok, x_dtype=2)), (4, dict(ok, x_pitch=k - 1)),
                     (4, dict(ok, y_pitch=n - 1)), (4, dict(ok, fault=None)), (40, dict(ok, workspace=None)), (40, dict(ok, workspace=ws[:-1])),
                     (40, dict(ok, workspace=ws[16:])), (49, ok), (40, dict(ok, workspace=ws.data_ptr()))):
        with pytest.raises(M.ExpertError) as e:
            M.linear_dev(layer, x, rows, y, **kw)
        assert e.value.code == 1
    for xx, yy in ((None, y), (x, None), (x.data_ptr() + 1, y), (x, y.data_ptr() + 2)):
        with pytest.raises(M.ExpertError) as e:
            M.linear_dev(layer, xx, 4, yy, **ok)
        assert e.value.code == 1
    torch.cuda.synchronize()
    assert layer.workspace_bytes(0) == 0 < layer.workspace_bytes(1) and layer.workspace_bytes(8192) == layer.workspace_bytes(1 << 20)


# --------------------------------------------------------------------------------------------------------------- norm
def norm_f64(planes, residual, post_w, gate, kind, pre_w, eps, ys, rs):
    u = sum(p.double() for p in planes) if planes else None
    if u is not None and post_w is not None:
        u = u / (u.square().mean(-1, keepdim=True) + eps).sqrt() * post_w.double()
    if kind == 1:
        u = u * gate.double()[:, None]
    elif kind:
        u = u * gate.double()
    h = 0 if u is None else ys * u
    if residual is not None:
        h = h + rs * residual.double()
    n = h / (h.square().mean(-1, keepdim=True) + eps).sqrt()
    return h, n if pre_w is None else n * pre_w.double()


def norm_case(torch, rows, width, *, planes=1, y32=False, h32=True, n32=True, w32=True, kind=0, post=True, pre=True, residual=True, in_place=False,
              pad=0, off=0, seed=0, scale=1.0):
    import mimo26f_afd_b200 as M

    g = gen(torch, seed + rows * 131 + width)
    ty = {True: torch.float32, False: torch.bfloat16}

    def buf(f32, fill=True):
        b = torch.full((off + (rows + 1) * (width + pad),), float("nan"), dtype=ty[f32], device="cuda")
        v = torch.as_strided(b, (rows, width), (width + pad, 1), off)
        if fill:
            v.copy_(scale * torch.randn(rows, width, device="cuda", generator=g))
        return b, v

    ys = [buf(y32)[1] for _ in range(planes)]
    res_b, res = buf(h32) if residual else (None, None)
    pw = torch.randn(width, device="cuda", generator=g).to(ty[w32]) if post and planes else None
    nw = torch.randn(width, device="cuda", generator=g).to(ty[w32]) if pre else None
    gate = None
    if kind == 1:
        gate = torch.randn(rows, device="cuda", generator=g)
    elif kind == 2:
        gate = torch.randn(width, device="cuda", generator=g).to(ty[w32])
    elif kind == 3:
        gate = buf(y32)[1]
    res0 = res.double().abs() if residual else None
    hb, h = (res_b, res) if in_place else buf(h32, False)
    nb, n = buf(n32, False)
    want_h, want_n = norm_f64(ys, res, pw, gate, kind, nw, 1e-5, 0.75, -1.5)
    M.block_norm_dev(ys, res, rows, width, post_w=pw, gate=gate, gate_kind=kind, y_dtype=int(y32), y_pitch=width + pad, y_scale=0.75, h_dtype=int(h32),
                     h_pitch=width + pad, residual_scale=-1.5, pre_w=nw, w_dtype=int(w32), eps=1e-5, h_out=h, n_out=n, n_dtype=int(n32), n_pitch=width + pad)
    torch.cuda.synchronize()
    # FP32: every term of h within 64 u of its own size; the sum of planes may cancel, so by the terms
    terms = 0.75 * sum(p.double().abs() for p in ys) if planes else torch.zeros_like(want_n)
    if planes and pw is not None:
        u = sum(p.double() for p in ys)
        terms = terms / (u.square().mean(-1, keepdim=True) + 1e-5).sqrt() * pw.double().abs()
    if kind:
        terms = terms * (gate.double().abs()[:, None] if kind == 1 else gate.double().abs())
    if residual:
        terms = terms + 1.5 * res0
    dh = 64 * U * terms
    eps_b = lambda f32: 0.0 if f32 else 2.0**-8  # noqa: E731
    assert bool(((h.double() - want_h).abs() <= dh + eps_b(h32) * (want_h.abs() + dh)).all())
    # n = h w / rms, so an error dh of h is |w| / rms dh of n (also where h itself is zero), beside that of the row's rms
    rms = (want_h.square().mean(-1, keepdim=True) + 1e-5).sqrt()
    r = (nw.double().abs() if nw is not None else 1.0) / rms
    mean_dh = (dh.square().mean(-1, keepdim=True)).sqrt() / rms
    dn = r * dh + (64 * U + mean_dh) * want_n.abs() + 1e-30
    assert bool(((n.double() - want_n).abs() <= dn + eps_b(n32) * (want_n.abs() + dn)).all())
    h.fill_(float("nan"))
    n.fill_(float("nan"))
    assert bool(torch.isnan(hb).all()) and bool(torch.isnan(nb).all())       # nothing outside the rows was written


@pytest.mark.parametrize("width", [1, 2, 7, 8, 31, 32, 33, 64, 255, 256, 257, 1000, 1024, 4095, 4096, 8192, 8200, 9999, 16384, 16392, 20001, 32767, 32768])
@pytest.mark.parametrize("rows", [1, 5])
def test_norm_widths(torch, rows, width):
    norm_case(torch, rows, width)


@pytest.mark.parametrize("width", [1, 2, 3, 5, 63, 255, 257, 1021, 1027, 4093, 4095, 5001, 8191, 16381, 20003, 32765])
@pytest.mark.parametrize("planes,kind", [(1, 3), (4, 1)])
def test_norm_odd_widths_in_aligned_rows(torch, width, planes, kind):
    """Rows on vector boundaries whose last vector is short."""
    norm_case(torch, 5, width, planes=planes, kind=kind, pad=-width % 4)
    norm_case(torch, 3, width, planes=planes, kind=kind, pad=-width % 8, h32=False, n32=False, w32=False)


@pytest.mark.parametrize("y32", [False, True])
@pytest.mark.parametrize("h32", [False, True])
@pytest.mark.parametrize("n32,w32", [(False, True), (True, False), (False, False)])
@pytest.mark.parametrize("width", [1024, 1023])
def test_norm_types(torch, y32, h32, n32, w32, width):
    norm_case(torch, 9, width, y32=y32, h32=h32, n32=n32, w32=w32, kind=3)


@pytest.mark.parametrize("kind", [0, 1, 2, 3])
@pytest.mark.parametrize("post", [False, True])
@pytest.mark.parametrize("pre", [False, True])
@pytest.mark.parametrize("width", [512, 77])
def test_norm_gates_and_optional_parts(torch, kind, post, pre, width):
    norm_case(torch, 6, width, kind=kind, post=post, pre=pre, planes=3)
    norm_case(torch, 6, width, kind=kind, post=post, pre=pre, residual=False)


@pytest.mark.parametrize("planes", [0, 1, 2, 3, 4, 5, 6, 7, 8])
def test_norm_planes(torch, planes):
    norm_case(torch, 4, 768, planes=planes, post=planes > 0)
    norm_case(torch, 4, 770, planes=planes, post=planes > 0)


@pytest.mark.parametrize("pad,off", [(0, 0), (8, 8), (3, 0), (0, 1), (16, 4), (4, 0)])
@pytest.mark.parametrize("in_place", [False, True])
def test_norm_strides_alignment_and_in_place(torch, pad, off, in_place):
    for h32 in (True, False):
        norm_case(torch, 7, 640, pad=pad, off=off, in_place=in_place, h32=h32, n32=False)


@pytest.mark.parametrize("rows", [2, 3, 4, 127, 1000, 5000])
def test_norm_rows(torch, rows):
    norm_case(torch, rows, 96)
    norm_case(torch, rows, 2048, h32=False, n32=False)


def test_norm_plane_sum_is_the_rank_sum(torch):
    """With nothing but planes and a residual, h is m26b_rank_sum_residual_dev's bits."""
    import mimo26f_afd_b200 as M

    rows, width = 5, 4096
    g = gen(torch, 3)
    planes = [torch.randn(rows, width, device="cuda", generator=g).to(torch.bfloat16) for _ in range(4)]
    res = torch.randn(rows, width, device="cuda", generator=g)
    want, h = torch.empty_like(res), torch.empty_like(res)
    M.rank_sum_dev(planes, rows * width, want, residual=res)
    M.block_norm_dev(planes, res, rows, width, h_out=h)
    torch.cuda.synchronize()
    assert torch.equal(h, want)


def test_norm_of_zero_huge_and_nonfinite_rows(torch):
    import mimo26f_afd_b200 as M

    for width in (256, 255):
        h = torch.zeros(6, width, device="cuda")
        h[1] = 1e-30
        h[2] = 3e38 * torch.where(torch.arange(width, device="cuda") % 2 == 0, 1.0, -1.0)
        h[3] = 1.0
        h[3, 5] = 1e25
        h[4] = 1.0
        h[4, 7] = float("inf")
        h[5] = 1.0
        h[5, 7] = float("nan")
        n = torch.empty_like(h)
        M.block_norm_dev([], h, 6, width, n_out=n, n_dtype=1, eps=1e-6)
        torch.cuda.synchronize()
        d = h.double()
        want = d / (d.square().mean(-1, keepdim=True) + 1e-6).sqrt()
        assert bool(((n.double() - want)[:4].abs() <= 64 * U * want[:4].abs()).all())
        assert bool(torch.isnan(n[4, 7])) and float(n[4].nan_to_num().abs().max()) == 0.0      # finite / inf = 0, inf / inf = NaN
        assert bool(torch.isnan(n[5]).all())


# ----------------------------------------------------------------------------------------------------------- together
def test_a_moe_block_with_a_shared_expert_between_two_norms(torch):
    """norm -> routed experts (m26b_ffn_dev) and a shared expert (gated, linear) -> their sum, the residual and the next norm, on one
    stream and replayed from a graph; the sum is m26b_rank_sum_residual_dev's bits, the shared expert is held to 64 bits."""
    import mimo26f_afd_b200 as M
    from mimo26f_afd_b200 import synth

    rows, H, I = 16, 4096, 2048
    dev = torch.device("cuda:0")
    g = gen(torch, 4)
    routed_w = synth.layer_torch(7, dev)
    layer = M.Layer.from_checkpoint(*[routed_w[n] for n in synth.TENSORS])
    shared = {n: routed_w[n][5] for n in synth.TENSORS}          # expert 5's tensors stand for the shared expert's
    up = M.Linear.gated(shared["gate_w"], shared["gate_s"], shared["up_w"], shared["up_s"], I, H)
    down = M.Linear.new(shared["down_w"], shared["down_s"], H, I)
    scratch = M.Scratch()
    ids, wts = (torch.from_numpy(np.ascontiguousarray(a)).cuda() for a in synth.routing(7, rows, 0.0))
    ws = torch.empty(max(up.workspace_bytes(rows), down.workspace_bytes(rows)), dtype=torch.uint8, device="cuda")
    fault = torch.zeros(1, dtype=torch.int32, device="cuda")
    h0 = torch.randn(rows, H, device="cuda", generator=g)
    w1, w2 = (1 + 0.1 * torch.randn(H, device="cuda", generator=g) for _ in range(2))
    h = torch.zeros_like(h0)
    n1, routed, y, n2 = (torch.zeros(rows, H, dtype=torch.bfloat16, device="cuda") for _ in range(4))
    a = torch.zeros(rows, I, dtype=torch.bfloat16, device="cuda")

    def step(st):
        M.block_norm_dev([], h0, rows, H, pre_w=w1, n_out=n1, stream=st)
        M.ffn_dev(layer, scratch, n1, ids, wts, rows, routed, stream=st)
        M.linear_dev(up, n1, rows, a, workspace=ws, fault=fault, stream=st)
        M.linear_dev(down, a, rows, y, workspace=ws, fault=fault, stream=st)
        M.block_norm_dev([routed, y], h0, rows, H, pre_w=w2, h_out=h, n_out=n2, stream=st)

    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    step(side.cuda_stream)
    scratch.status(side.cuda_stream)
    torch.cuda.synchronize()
    first = [t.clone() for t in (n1, routed, a, y, h, n2)]
    want = torch.empty_like(h0)
    M.rank_sum_dev([routed, y], rows * H, want, residual=h0)
    torch.cuda.synchronize()
    assert torch.equal(h, want)
    _, nn = norm_f64([], h, None, None, 0, w2, 1e-6, 1.0, 1.0)
    assert bool(((n2.double() - nn).abs() <= (2.0**-8 + 64 * U) * nn.abs()).all())
    G, Up, D = (weight_f64(torch, shared[p + "_w"], shared[p + "_s"]) for p in ("gate", "up", "down"))
    p, dp = product_and_bound(torch, n1.double(), G)
    q, dq = product_and_bound(torch, n1.double(), Up)
    silu = p * torch.sigmoid(p)
    check(torch, a, silu * q, rounded(silu * q, 1.1 * dp * (q.abs() + dq) + silu.abs() * dq + 2.0**-19 * (silu * q).abs(), True))
    z, dz = product_and_bound(torch, a.double(), D)
    check(torch, y, z, rounded(z, dz, True))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        step(side.cuda_stream)
    for t in (n1, routed, a, y, h, n2):
        t.zero_()
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(u, v) for u, v in zip(first, (n1, routed, a, y, h, n2))) and int(fault) == 0


@pytest.mark.parametrize("rows", [1, 16, 140])
def test_a_dense_block_between_two_norms(torch, rows):
    """norm -> gated -> linear -> norm, as a dense block of a decoder runs them: captured once and replayed, against 64 bits
    through every BF16 rounding of the chain."""
    import mimo26f_afd_b200 as M

    H, I = 1024, 1536
    g = gen(torch, rows)
    gw, gs = make_weights(torch, I, H, g)
    uw, us = make_weights(torch, I, H, g)
    dw, ds = make_weights(torch, H, I, g)
    up, down = M.Linear.gated(gw, gs, uw, us, I, H), M.Linear.new(dw, ds, H, I)
    ws = torch.empty(max(up.workspace_bytes(rows), down.workspace_bytes(rows)), dtype=torch.uint8, device="cuda")
    fault = torch.zeros(1, dtype=torch.int32, device="cuda")
    h0 = torch.randn(rows, H, device="cuda", generator=g)
    w1, w2, w3 = (1 + 0.1 * torch.randn(H, device="cuda", generator=g) for _ in range(3))
    h = torch.empty_like(h0)
    n1, n2, y = (torch.empty(rows, H, dtype=torch.bfloat16, device="cuda") for _ in range(3))
    a = torch.empty(rows, I, dtype=torch.bfloat16, device="cuda")

    def step(st):
        M.block_norm_dev([], h0, rows, H, pre_w=w1, n_out=n1, stream=st)
        M.linear_dev(up, n1, rows, a, workspace=ws, fault=fault, stream=st)
        M.linear_dev(down, a, rows, y, workspace=ws, fault=fault, stream=st)
        M.block_norm_dev([y], h0, rows, H, post_w=w2, pre_w=w3, h_out=h, n_out=n2, stream=st)

    step(None)
    torch.cuda.synchronize()
    first = [t.clone() for t in (n1, a, y, h, n2)]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(torch.cuda.current_stream().cuda_stream)
    for t in (n1, a, y, h, n2):
        t.zero_()
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(first, (n1, a, y, h, n2)))
    assert int(fault) == 0
    # each stage from the stored input of that stage
    _, want = norm_f64([], h0, None, None, 0, w1, 1e-6, 1.0, 1.0)
    assert bool(((n1.double() - want).abs() <= (2.0**-8 + 128 * U) * want.abs()).all())
    p, dp = product_and_bound(torch, n1.double(), weight_f64(torch, gw, gs))
    q, dq = product_and_bound(torch, n1.double(), weight_f64(torch, uw, us))
    silu = p * torch.sigmoid(p)
    check(torch, a, silu * q, rounded(silu * q, 1.1 * dp * (q.abs() + dq) + silu.abs() * dq + 2.0**-19 * (silu * q).abs(), True))
    z, dz = product_and_bound(torch, a.double(), weight_f64(torch, dw, ds))
    check(torch, y, z, rounded(z, dz, True))
    hh, nn = norm_f64([y], h0, w2, None, 0, w3, 1e-6, 1.0, 1.0)
    assert bool(((h.double() - hh).abs() <= 128 * U * (h0.double().abs() + (hh - h0.double()).abs())).all())
    rms = (hh.square().mean(-1, keepdim=True) + 1e-6).sqrt()
    dn = 128 * U * ((h0.double().abs() + (hh - h0.double()).abs()) / rms * w3.double().abs() + nn.abs())
    assert bool(((n2.double() - nn).abs() <= dn + 2.0**-8 * (nn.abs() + dn)).all())
