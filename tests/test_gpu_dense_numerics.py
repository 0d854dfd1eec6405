"""The dense operators where FP32 itself decides: sums that are exact by construction, the activation over the whole range of its
argument, norm factors near the ends of the range. Formulas in 64 bits; helpers and the derivation of the common bounds are
test_gpu_dense's."""
import pytest
import test_gpu_dense as D

pytestmark = pytest.mark.gpu

U = D.U


@pytest.fixture(scope="module")
def torch():
    import torch

    assert torch.cuda.is_available(), "these tests need the GPU box"
    return torch


@pytest.mark.parametrize("rows,n,k,fine,split", [(20, 200, 512, 7, 8), (300, 1000, 1024, 6, 8), (2048, 4096, 4096, 4, 1), (300, 4096, 16384, 2, 1), (273, 11344, 2048, 5, 1)])
@pytest.mark.parametrize("gated", [False, True])
def test_sums_that_fit_fp32_are_exact(torch, rows, n, k, fine, split, gated):
    """Activations 128..255 (eight significant bits), weights 0.5 and mostly 6, every other K32 block scaled by 2^-fine. The leading pieces'
    products are multiples of 8 * 2^-fine and their sums fit 24 bits, the second pieces' are multiples of 2^-fine / 2 and theirs fit too: both
    are exact in FP32, so what comes out is the true sum, rounded once. As one running sum they would need 26 bits and lose some
    in every step. Gated: a gate of 256 makes the activation the identity (e^-256 is nothing beside 1)."""
    import mimo26f_afd_b200 as M

    step = 2.0**-fine
    assert k / 2 * 6 * 256 * (1 + step) < 2**24 * 8 * step and k * 6 * 8 < 2**24 * step / 2     # 256: a leading piece rounds up to it
    g = D.gen(torch, rows + k)
    x = torch.randint(128, 256, (rows, k), device="cuda", generator=g)
    x[:, ::32] = 255
    x = x.to(torch.bfloat16)
    w = torch.where(torch.rand(n, k, device="cuda", generator=g) < 0.1, 1, 7).to(torch.uint8)            # E2M1 codes of 0.5 and 6
    w = w[:, 0::2] | w[:, 1::2] << 4
    s = torch.full((n, k // 32), 127, dtype=torch.uint8, device="cuda")
    s[:, 1::2] -= fine
    want = x.double() @ D.weight_f64(torch, w, s).T                        # exact in 64 bits
    layer = M.Linear.new(w, s, n, k)
    if gated:
        gw = torch.zeros_like(w)                                           # one weight of 1 on the block's first activation: 255
        gw[:, 0] = 2
        layer = M.Linear.gated(gw, torch.full_like(s, 127), w, s, n, k)
        want = want * 255
    run = D.Runner(torch, layer, rows)
    y = run(x, rows)
    torch.cuda.synchronize()
    ulp = torch.exp2(torch.floor(torch.log2(want)) - 23)
    # half a unit; where K is split (at most eight ways), one for each partial result and one for each sum of two; the activation 4 units
    allowed = (2 * split - 1) / 2 + (4 if gated else 0)
    off = (y.double() - want).abs() / ulp
    assert float(off.max()) <= allowed, f"{float(off.max()):.3g} units in the last place"
    assert int(run.fault) == 0


@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("rows,n,k", [(100, 4096, 16384), (100, 20000, 4096), (2048, 4096, 4096), (700, 9600, 4096)])
def test_a_wait_that_runs_out_is_reported(torch, rows, n, k, gated):
    """A bound of a microsecond on accumulators that take ten and more: K split over a cluster, single CTAs, CTA pairs with one and with several
    items each. The kernel ends, the fault word says so, and the handle works on."""
    import mimo26f_afd_b200 as M

    g = D.gen(torch, rows)
    w, s = D.make_weights(torch, n, k, g)
    layer = M.Linear.gated(w, s, w, s, n, k) if gated else M.Linear.new(w, s, n, k)
    x = torch.randn(rows, k, device="cuda", generator=g).to(torch.bfloat16)
    run = D.Runner(torch, layer, rows)
    want = run(x, rows).clone()
    torch.cuda.synchronize()
    assert int(run.fault) == 0
    layer.set_wait_us(1)
    run(x, rows)
    torch.cuda.synchronize()
    assert int(run.fault) == 3
    layer.set_wait_us(200_000)
    run.fault.zero_()
    got = run(x, rows)
    torch.cuda.synchronize()
    assert int(run.fault) == 0 and torch.equal(got, want)


@pytest.mark.parametrize("width", [256, 255, 1000, 4096, 4095, 16384])
@pytest.mark.parametrize("kind", [0, 1, 2, 3])
@pytest.mark.parametrize("post", [False, True])
def test_factors_that_fp32_cannot_hold_as_one(torch, width, kind, post):
    """Rows of every size FP32 has, with a scale and a gate whose product with the row's 1 / rms lies below its range although the
    result is ordinary. Every product of two factors is a rounding: 64 u as everywhere."""
    import mimo26f_afd_b200 as M

    g = D.gen(torch, width + kind)
    size = torch.tensor([1e38, 1e38, 1e30, 1e20, 1.0, 1e-10, 1e-18], device="cuda")
    rows = len(size)
    u = (0.25 + 0.75 * torch.rand(rows, width, device="cuda", generator=g)) * size[:, None]
    u = torch.where(torch.rand(rows, width, device="cuda", generator=g) < 0.5, -u, u)
    pw = 0.5 + torch.rand(width, device="cuda", generator=g) if post else None
    # gates that bring the largest rows down where no norm does
    weight = torch.tensor([1e-6, 1e-10, 1e-16, 1e-4, 1.0, 1e4, 0.0], device="cuda") * (1.0 if post else 1e-6)
    gate = None
    if kind == 1:
        gate = weight
    elif kind == 2:
        gate = 1e-6 + 1e-6 * torch.rand(width, device="cuda", generator=g)
    elif kind == 3:
        gate = weight[:, None] * (0.5 + torch.rand(rows, width, device="cuda", generator=g))
    for ys in (1e-12, 1e-3, -1.0) if post else (1e-25, 1e-12, -1.0):
        h, n = torch.empty_like(u), torch.empty_like(u)
        M.block_norm_dev([u], None, rows, width, post_w=pw, gate=gate, gate_kind=kind, y_dtype=1, y_scale=ys, h_out=h, n_out=n, n_dtype=1, eps=1e-6)
        torch.cuda.synchronize()
        scale = float(torch.tensor(ys, dtype=torch.float32))
        want, wn = D.norm_f64([u], None, pw, gate, kind, None, float(torch.tensor(1e-6, dtype=torch.float32)), scale, 1.0)
        keep = want.abs() >= 2.0**-120                          # below, the result itself runs out of bits
        assert bool(((h.double() - want).abs() <= 64 * U * want.abs() + 2.0**-149)[keep].all())
        assert bool((h.double()[~keep].abs() <= 2.0**-119).all())
        assert bool(((n.double() - wn).abs() <= 128 * U * wn.abs())[keep].all())


@pytest.mark.parametrize("width", [256, 255, 4096, 4095, 16384])
def test_norms_of_rows_near_the_bottom_of_fp32(torch, width):
    """Squares that FP32 holds in part or not at all, beside the smallest eps that the norm takes."""
    import mimo26f_afd_b200 as M

    g = D.gen(torch, width)
    for eps in (2.0**-126, 1e-36, 1e-30, 1e-20, 1e-6):
        size = torch.tensor([1e-22, 1e-20, 1e-19, 1e-16, 1e-12, 1.0, 1e30], device="cuda")
        h = (torch.rand(len(size), width, device="cuda", generator=g) - 0.5) * size[:, None]
        n = torch.empty_like(h)
        M.block_norm_dev([], h, len(size), width, n_out=n, n_dtype=1, eps=eps)
        torch.cuda.synchronize()
        _, want = D.norm_f64([], h, None, None, 0, None, float(torch.tensor(eps, dtype=torch.float32)), 1.0, 1.0)
        assert bool(((n.double() - want).abs() <= 64 * U * want.abs() + 2.0**-149).all()), eps
