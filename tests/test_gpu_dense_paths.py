"""The dense operators' kernels, each reached on purpose: CTA pairs with every kind of token tile, from rows in place and staged, and the
norm's rows beyond those that run at once, with everything that is fetched ahead. Bounds and helpers are test_gpu_dense's."""
import pytest
import test_gpu_dense as D
from test_dense_rules import PAIR_SHAPES

pytestmark = pytest.mark.gpu

IDS = ["%s-%s-%dx%d-%d-tile%d" % ("bf16" if b else "e4m3", "gated" if g else "linear", n, k, r, t) for b, g, n, k, r, t in PAIR_SHAPES]


@pytest.fixture(scope="module")
def torch():
    import torch

    assert torch.cuda.is_available(), "these tests need the GPU box"
    return torch


def strided(torch, rows, k, pad, off, dtype, fill):
    """[rows, k] in a buffer whose other elements are `fill`."""
    buf = torch.full((off + rows * (k + pad),), fill, dtype=dtype, device="cuda")
    return torch.as_strided(buf, (rows, k), (k + pad, 1), off)


@pytest.mark.parametrize("bf16,gated,n,k,rows,tile", PAIR_SHAPES, ids=IDS)
def test_pairs(torch, bf16, gated, n, k, rows, tile):
    """Both output types into padded rows, activations on 16-byte boundaries and on odd ones (E4M3: in place, staged as vectors, staged byte
    by byte)."""
    import mimo26f_afd_b200 as M

    g = D.gen(torch, n + k + rows)
    mats = [D.make_weights(torch, n, k, g) for _ in range(1 + gated)]
    W = [D.weight_f64(torch, *m) for m in mats]
    layer = M.Linear.gated(*mats[0], *mats[1], n, k) if gated else M.Linear.new(*mats[0], n, k)
    run = D.Runner(torch, layer, rows)
    scales = None
    if bf16:
        data = torch.randn(rows, k, device="cuda", generator=g).to(torch.bfloat16)
        values = data.double()
    else:
        data = torch.randint(0, 256, (rows, k), dtype=torch.uint8, device="cuda", generator=g)
        data[(data & 127) == 127] = 0x38
        scales = torch.randint(112, 118, (rows, k // 32), dtype=torch.uint8, device="cuda", generator=g)
        if gated:
            scales -= 6                                           # keep the activation's argument moderate
        values = D.e4m3_f64(torch, data, scales)
    y, bound = D.product_and_bound(torch, values, W[0], quantised=not bf16)
    if gated:
        b, db = D.product_and_bound(torch, values, W[1], quantised=not bf16)
        silu = y * torch.sigmoid(y)
        bound = 1.1 * bound * (b.abs() + db) + silu.abs() * db + 2.0**-19 * (silu * b).abs()
        y = silu * b
    del W
    first = None
    for pad, off in ((0, 0), (8, 0), (3, 1)):
        x = strided(torch, rows, k, pad, off, data.dtype, float("nan") if bf16 else 0x7f)
        x.copy_(data)
        for f32 in (True, False):
            yb = torch.full(((rows + 1) * (n + 5),), -77.0, dtype=torch.float32 if f32 else torch.bfloat16, device="cuda")
            out = torch.as_strided(yb, (rows, n), (n + 5, 1), 0)
            run(x, rows, f32=f32, x_scales=scales, x_pitch=k + pad, y=out, y_pitch=n + 5)
            D.check(torch, out, y, D.rounded(y, bound, not f32))
            if f32:
                first = out.clone() if first is None else first
                assert torch.equal(out, first)                    # however the rows arrive
            out.fill_(-77.0)
            assert bool((yb == -77.0).all())                      # nothing outside the rows was written
    assert int(run.fault) == 0


@pytest.mark.parametrize("pad", [0, 8, 3])
@pytest.mark.parametrize("bf16", [False, True])
def test_nonfinite_rows_on_pairs(torch, pad, bf16):
    import mimo26f_afd_b200 as M

    n, k, rows = (1549, 32, 4038) if bf16 else (14409, 128, 395)
    layer = M.Linear.new(*D.make_weights(torch, n, k, D.gen(torch, 4)), n, k)
    bad = (1, 2, 130, 394)
    if bf16:
        x = strided(torch, rows, k, pad, 0, torch.bfloat16, 0.0)
        x.fill_(1.0)
        x[1, 5], x[2, 31], x[130, 0], x[394, 7] = float("nan"), float("inf"), float("-inf"), float("nan")
        xs = None
    else:
        x = strided(torch, rows, k, pad, 0, torch.uint8, 0)
        x.fill_(0x38)
        xs = torch.full((rows, k // 32), 127, dtype=torch.uint8, device="cuda")
        x[1, 40], x[2, 127] = 0x7f, 0xff
        xs[130, 3], xs[394, 0] = 255, 255
    y = D.Runner(torch, layer, rows)(x, rows, x_scales=xs, x_pitch=k + pad)
    torch.cuda.synchronize()
    nan = torch.isnan(y)
    want = [i in bad for i in range(rows)]
    assert nan.all(1).tolist() == want and nan.any(1).tolist() == want


@pytest.mark.parametrize("rows,width,pad", [(20000, 256, 0), (5000, 1000, 0), (5000, 1024, 8), (5000, 1021, 3), (3000, 4096, 0), (3000, 4093, 3), (3000, 4093, 0), (1500, 8192, 0)])
@pytest.mark.parametrize("kind,planes", [(3, 1), (3, 3), (1, 8), (2, 2)])
def test_norm_of_more_rows_than_run_at_once(torch, rows, width, pad, kind, planes):
    """Every CTA takes several rows and fetches the next one's planes, residual and gate while it reduces this one's."""
    for h32 in (False, True):
        for in_place in (False, True):
            D.norm_case(torch, rows, width, planes=planes, kind=kind, h32=h32, n32=h32, in_place=in_place, pad=pad, seed=planes)


@pytest.mark.parametrize("rows,width,pad", [(5000, 1024, 0), (5000, 1021, 3), (5000, 1021, 0)])
@pytest.mark.parametrize("kind", [0, 3])
def test_norm_of_fp32_planes_and_of_no_planes_beyond_one_round(torch, rows, width, pad, kind):
    D.norm_case(torch, rows, width, y32=True, kind=kind, pad=pad, in_place=True)
    D.norm_case(torch, rows, width, y32=True, kind=kind, pad=pad, h32=False, w32=False)
    D.norm_case(torch, rows, width, planes=0, pad=pad)
    D.norm_case(torch, rows, width, planes=0, pad=pad, h32=False, in_place=True)
