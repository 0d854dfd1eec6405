"""The dense operators' argument checks, which come before any CUDA call."""
import ctypes

import pytest

P = 0x10000          # a device address that is never touched: every call here is refused, or has no rows


def block_norm(**kw):
    import mimo26f_afd_b200 as M

    a = dict(planes=[P], residual=P, rows=0, width=64, h_out=P, n_out=P)
    a.update(kw)
    M.block_norm_dev(a.pop("planes"), a.pop("residual"), a.pop("rows"), a.pop("width"), **a)


def test_block_norm_without_rows_is_no_work():
    block_norm()
    block_norm(planes=[])
    block_norm(planes=[P] * 8, residual=None, post_w=P, gate=P, gate_kind=3, pre_w=P)
    block_norm(n_out=None)
    block_norm(h_out=None, width=32768)


@pytest.mark.parametrize("kw", [
    dict(width=0), dict(width=32769), dict(planes=[P] * 9), dict(planes=[P, 0]), dict(planes=[], residual=None),
    dict(planes=[], post_w=P), dict(planes=[], gate=P, gate_kind=1), dict(gate=P), dict(gate_kind=2), dict(gate=P, gate_kind=4),
    dict(gate=P, gate_kind=-1), dict(y_dtype=2), dict(h_dtype=-1), dict(n_dtype=2), dict(w_dtype=3), dict(h_out=None, n_out=None),
    dict(n_out=None, pre_w=P), dict(eps=0.0), dict(eps=-1e-6), dict(eps=float("nan")), dict(eps=float("inf")),
    dict(rows=1 << 31), dict(y_pitch=63), dict(h_pitch=63), dict(n_pitch=1),
    dict(planes=[P + 1]), dict(planes=[P + 2], y_dtype=1), dict(residual=P + 2), dict(n_out=P + 1), dict(pre_w=P + 2),
    dict(gate=P + 2, gate_kind=1), dict(gate=P + 1, gate_kind=3),
])
def test_block_norm_refuses(kw):
    import mimo26f_afd_b200 as M

    with pytest.raises(M.ExpertError) as e:
        block_norm(**kw)
    assert e.value.code == 1 and "m26b block norm" in e.value.message


@pytest.mark.parametrize("kw", [dict(rows=-1), dict(rows=1 << 32), dict(y_pitch=-64), dict(gate_kind=1 << 40)])
def test_numbers_that_do_not_fit_the_record_are_refused(kw):
    import mimo26f_afd_b200 as M

    with pytest.raises(M.ExpertError) as e:
        block_norm(**kw)
    assert e.value.code == 1

    class Handle:
        _h = None

    with pytest.raises(M.ExpertError) as e:
        M.linear_dev(Handle(), P, kw.get("rows", -1), P)
    assert e.value.code == 1


def test_argument_records_match_the_header():
    """Sizes of the packed records against the C structs, compiled here."""
    import subprocess
    import tempfile

    from conftest import ROOT
    from mimo26f_afd_b200 import dense

    with tempfile.TemporaryDirectory() as d:
        src = f'{d}/sizes.c'
        with open(src, "w") as f:
            f.write('#include <stdio.h>\n#include <stddef.h>\n#include "m26b_expert.h"\nint main(void) { printf("%zu %zu %zu %zu %zu %zu\\n", '
                    'sizeof(m26b_linear_args), offsetof(m26b_linear_args, rows), offsetof(m26b_linear_args, x_pitch), '
                    'sizeof(m26b_block_norm_args), offsetof(m26b_block_norm_args, y_scale), offsetof(m26b_block_norm_args, n_planes)); return 0; }')
        subprocess.run(["gcc", "-I", f"{ROOT}/include", "-o", f"{d}/sizes", src], check=True)
        got = [int(v) for v in subprocess.run([f"{d}/sizes"], check=True, capture_output=True, text=True).stdout.split()]
    assert got[0] == (dense._LINEAR_ARGS.size + 7) // 8 * 8 and got[1] == 64 and got[2] == 48
    assert got[3] == (dense._NORM_ARGS.size + 7) // 8 * 8 and got[4] == 14 * 8 + 3 * 8 and got[5] == got[4] + 20


@pytest.mark.parametrize("n,k", [(0, 64), (64, 0), (64, 33), (64, 16), ((1 << 20) + 1, 64), (64, (1 << 20) + 32)])
def test_linear_refuses_extents(n, k):
    import mimo26f_afd_b200 as M

    for make in (lambda: M.Linear.new(P, P, n, k), lambda: M.Linear.gated(P, P, P, P, n, k)):
        with pytest.raises(M.ExpertError) as e:
            make()
        assert e.value.code == 1 and "m26b linear" in e.value.message


def test_linear_refuses_null_tensors_and_handles():
    import mimo26f_afd_b200 as M
    from mimo26f_afd_b200 import _native

    for make in (lambda: M.Linear.new(None, P, 64, 64), lambda: M.Linear.new(P, None, 64, 64), lambda: M.Linear.gated(P, P, None, P, 64, 64),
                 lambda: M.Linear.gated(P, P, P, None, 64, 64)):
        with pytest.raises(M.ExpertError) as e:
            make()
        assert e.value.code == 1
    lib = _native.lib()
    err = ctypes.create_string_buffer(256)
    at = ctypes.addressof(err)
    assert lib.m26b_linear_dev(None, b"\0" * 256, None, at, 256) == 1 and b"bad handle" in err.value
    assert lib.m26b_block_norm_dev(None, None, at, 256) == 1 and b"bad arguments" in err.value
    assert lib.m26b_linear_workspace_bytes(None, 5) == 0
    lib.m26b_linear_free(None)


def test_linear_without_a_gpu_fails_loudly():
    import torch

    if torch.cuda.is_available():
        pytest.skip("a GPU is present")
    import mimo26f_afd_b200 as M

    with pytest.raises(M.ExpertError) as e:
        M.Linear.new(P, P, 64, 64)
    assert e.value.code == 2
