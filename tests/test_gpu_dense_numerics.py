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


@pytest.mark.parametrize("rows,n", [(24, 64), (100, 4100), (130, 64), (2000, 9600)])
def test_the_activation_over_the_whole_range_of_its_argument(torch, rows, n):
    """One gate weight and one up weight per feature, both 1: y = silu(x[0]) * x[32]. Two exponentials of half the argument (2 units each, met
    twice), a quotient (2 units) and three products: within 2^-19 of the result for every gate, as far as FP32 reaches."""
    import mimo26f_afd_b200 as M

    k = 64
    weight = torch.zeros(n, k // 2, dtype=torch.uint8, device="cuda")
    gw, uw = weight.clone(), weight.clone()
    gw[:, 0], uw[:, 16] = 2, 2
    s = torch.full((n, k // 32), 127, dtype=torch.uint8, device="cuda")
    g = D.gen(torch, rows)
    size = torch.exp2(torch.rand(rows, device="cuda", generator=g) * 20 - 10)
    size[:12] = torch.tensor([60.0, 70, 80, 88, 90, 95, 100, 103.5, 110, 140, 170, 3e38], device="cuda")
    sign = torch.where(torch.arange(rows, device="cuda") % 3 == 0, 1.0, -1.0)
    sign[:12] = -1.0
    x = torch.zeros(rows, k, dtype=torch.bfloat16, device="cuda")
    x[:, 0] = size * sign
    for up in (1.0, -1e30, 1e38):
        x[:, 32] = up
        run = D.Runner(torch, M.Linear.gated(gw, s, uw, s, n, k), rows)
        a = x[:, 0].double()
        want = (a * torch.sigmoid(a) * x[:, 32].double())[:, None].expand(rows, n)
        keep = want.abs() < 3.4e38
        y = run(x, rows)
        torch.cuda.synchronize()
        off = (y.double() - want).abs()
        assert bool((off <= 2.0**-19 * want.abs() + 2.0**-126 * 2.0**-19)[keep].all()), float((off / want.abs().clamp_min(2.0**-126))[keep].max()) * 2**19
        assert torch.equal(y[~keep], want.float()[~keep])


@pytest.mark.parametrize("rows", [5, 130])
@pytest.mark.parametrize("quantised", [False, True])
def test_gate_sums_beyond_fp32(torch, rows, quantised):
    """-inf gives -0 * u, as every gate below some -200 does; +inf gives inf * u."""
    import mimo26f_afd_b200 as M

    n, k = 64, 64
    gw, uw = (torch.zeros(n, k // 2, dtype=torch.uint8, device="cuda") for _ in range(2))
    gw[:, 0], uw[:, 16] = 7, 2
    gs, us = (torch.full((n, k // 32), b, dtype=torch.uint8, device="cuda") for b in (154, 127))
    run = D.Runner(torch, M.Linear.gated(gw, gs, uw, us, n, k), rows)
    if quantised:                                                # gates of 6 * 2^27 * 448 * 2^100
        q = torch.zeros(rows, k, dtype=torch.uint8, device="cuda")
        q[:, 32] = 0x44                                          # 3
        q[0::2, 0], q[1::2, 0] = 0xfe, 0x7e
        xs = torch.full((rows, k // 32), 127, dtype=torch.uint8, device="cuda")
        xs[:, 0] = 227
        y = run(q, rows, x_scales=xs)
    else:                                                        # gates of 6 * 2^27 * 1e30 = 8e38
        x = torch.zeros(rows, k, dtype=torch.bfloat16, device="cuda")
        x[:, 32] = 3.0
        x[0::2, 0], x[1::2, 0] = -1e30, 1e30
        y = run(x, rows)
    torch.cuda.synchronize()
    assert bool((y[0::2] == 0.0).all()) and bool((y[1::2] == float("inf")).all())


def test_far_gates_of_other_rows_change_nothing(torch):
    """The exact form for far gates is a choice per element: not of the rows beside it, nor of what pads the tile."""
    import mimo26f_afd_b200 as M

    n, k, rows = 320, 256, 37
    g = D.gen(torch, 21)
    gw, gs = D.make_weights(torch, n, k, g)
    uw, us = D.make_weights(torch, n, k, g)
    x = torch.randn(rows, k, device="cuda", generator=g).to(torch.bfloat16)
    run = D.Runner(torch, M.Linear.gated(gw, gs, uw, us, n, k), rows)
    want = run(x, rows).clone()
    x2 = x.clone()
    x2[1::2] *= 1000.0
    got = run(x2, rows)
    torch.cuda.synchronize()
    assert torch.equal(got[0::2], want[0::2])


def test_an_unaligned_fault_word_is_refused(torch):
    import mimo26f_afd_b200 as M

    n, k = 64, 64
    layer = M.Linear.new(*D.make_weights(torch, n, k, D.gen(torch, 1)), n, k)
    x, y = torch.zeros(4, k, dtype=torch.bfloat16, device="cuda"), torch.zeros(4, n, device="cuda")
    ws, f = torch.empty(layer.workspace_bytes(4), dtype=torch.uint8, device="cuda"), torch.zeros(2, dtype=torch.int32, device="cuda")
    for off in (1, 2, 3):
        with pytest.raises(M.ExpertError) as e:
            M.linear_dev(layer, x, 4, y, y_dtype=1, workspace=ws, fault=f.data_ptr() + off)
        assert e.value.code == 1
    M.linear_dev(layer, x, 4, y, y_dtype=1, workspace=ws, fault=f.data_ptr() + 4)
    torch.cuda.synchronize()
    assert f.tolist() == [0, 0]


def test_handles_made_by_several_threads_run_the_same_kernels(torch):
    """What a handle knows of the device does not depend on who else asks: the same K split, so the same bits."""
    import threading

    import mimo26f_afd_b200 as M

    n, k, rows = 256, 4096, 9
    g = D.gen(torch, 30)
    w, s = D.make_weights(torch, n, k, g)
    x = torch.randn(rows, k, device="cuda", generator=g).to(torch.bfloat16)
    want = D.Runner(torch, M.Linear.new(w, s, n, k), rows)(x, rows)
    torch.cuda.synchronize()
    layers = [[] for _ in range(8)]

    def make(to):
        for _ in range(20):
            to.append(M.Linear.new(w, s, n, k))

    threads = [threading.Thread(target=make, args=(to,)) for to in layers]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for layer in sum(layers, []):
        assert torch.equal(D.Runner(torch, layer, rows)(x, rows), want)
