"""The dense operators' host side beyond the argument checks: bounds, sizes and the choice of kernel."""
import pytest


def test_the_wait_bound_is_checked():
    import mimo26f_afd_b200 as M
    from mimo26f_afd_b200 import _native

    assert _native.lib().m26b_linear_set_wait_us(None, 5) == 1

    class Handle(M.Linear):
        def __init__(self):
            self._h = None

    for us in (-1, 0, 1 << 32, 5):                              # 5: no handle
        with pytest.raises(M.ExpertError) as e:
            Handle().set_wait_us(us)
        assert e.value.code == 1


@pytest.fixture(scope="module")
def rules(tmp_path_factory):
    """linear_rules.h, compiled for the host."""
    import ctypes as C
    import subprocess

    from conftest import ROOT

    d = tmp_path_factory.mktemp("rules")
    (d / "rules.cpp").write_text('''#include "linear_rules.h"
using namespace m26b;
extern "C" {
uint64_t workspace(uint32_t k_pad, uint32_t rows) { return linear_workspace(k_pad, rows); }
uint64_t blocks(uint32_t rows, uint32_t tile, uint32_t pieces) { return linear_scale_blocks(rows, tile, pieces); }
static LinearShape shape(uint32_t tiles, uint32_t chunks, const uint32_t* place) {          // place: SMs, room[2][4]
    LinearShape s{tiles, chunks, place[0], {}};
    for (int i = 0; i < 8; ++i) s.room[i / 4][i % 4] = place[1 + i];
    return s;
}
uint32_t pair_tile(uint32_t tiles, uint32_t chunks, const uint32_t* place, uint32_t ctas, int bf16, uint32_t rows) { return linear_pair_tile(shape(tiles, chunks, place), ctas, bf16, rows); }
uint32_t log_split(uint32_t tiles, uint32_t chunks, const uint32_t* place, uint64_t ctas, uint32_t per_sm) { return linear_log_split(shape(tiles, chunks, place), ctas, per_sm, chunks); }
uint32_t direct(uint32_t tiles, uint32_t chunks, const uint32_t* place, int bf16, uint32_t rows) { return linear_direct(shape(tiles, chunks, place), bf16, rows); }
uint32_t widest(int bf16) { return linear_widest_pair_tile(bf16); }
}
''')
    subprocess.run(["g++", "-std=c++17", "-O1", "-shared", "-fPIC", "-I", f"{ROOT}/mimo26f_afd_b200/csrc", "-o", str(d / "rules.so"), str(d / "rules.cpp")], check=True)
    lib = C.CDLL(str(d / "rules.so"))
    lib.workspace.restype = lib.blocks.restype = C.c_uint64
    for f in (lib.pair_tile, lib.widest, lib.log_split, lib.direct):
        f.restype = C.c_uint32
    lib.log_split.argtypes = [C.c_uint32, C.c_uint32, C.c_void_p, C.c_uint64, C.c_uint32]
    lib.b200 = (C.c_uint32 * 9)(148, 148, 148, 132, 120, 296, 296, 284, 264)       # as a B200 answers
    return lib


def test_every_token_tile_fits_the_workspace(rules):
    """Not only the tiles that the costs choose: the codes of both pieces and, behind them, the last scale block that the staging kernel writes and
    the last that a tensor map covers, for every number of tokens and every tile a kernel can run."""
    import numpy as np

    chunks = 3
    k_pad = 128 * chunks
    last = 0
    sizes = []
    for rows in range(1, 8193):
        size = rules.workspace(k_pad, rows)
        assert size >= last
        last = size
        sizes.append(size)
    assert rules.workspace(k_pad, 0) == 0 and rules.workspace(k_pad, 1 << 20) == last
    sizes = np.array(sizes)
    rows = np.arange(1, 8193)
    for pieces in (1, 2):
        codes = pieces * ((rows + 15) // 16 * 16) * k_pad
        for tile in range(64, rules.widest(pieces == 2) + 1, 16):
            runs = 2 if tile > 128 else 1
            used = rows > 64 if tile != 64 else rows > 0          # up to 64 tokens always take tiles of 64
            covered = np.array([rules.blocks(int(r), tile, pieces) for r in rows]) * chunks
            t, r = (rows - 1) // tile, (rows - 1) % tile          # place of the last token's scales, as linear_split_kernel computes it
            joint = rows <= 64
            written = np.where(joint, chunks, (t * chunks + chunks - 1) * runs * pieces + (r >> 7) * pieces + pieces)
            assert (written <= covered)[used].all()
            assert (codes + covered * 512 <= sizes)[used].all(), (pieces, tile)


def test_the_chosen_tiles_are_tiles_of_the_kernel(rules):
    import random

    rng = random.Random(7)
    for _ in range(20000):
        bf16, rows = rng.random() < 0.5, int(2 ** rng.uniform(0, 13))
        tile = rules.pair_tile(2 * int(2 ** rng.uniform(0, 9)), int(2 ** rng.uniform(0, 8)), rules.b200, 148, bf16, rows)
        assert tile == 0 or (rows > 128 and tile % 16 == 0 and 64 <= tile <= rules.widest(bf16))
    assert rules.pair_tile(32, 32, rules.b200, 0, 1, 2048) == 0            # a device that cannot place a pair


@pytest.mark.parametrize("eps", [1e-45, 1e-42, 1.17e-38])
def test_a_subnormal_eps_is_refused(eps):
    """Rows as small as its root have squares that FP32 cannot hold beside it."""
    import mimo26f_afd_b200 as M

    p = 0x10000
    with pytest.raises(M.ExpertError) as e:
        M.block_norm_dev([p], p, 0, 64, h_out=p, n_out=p, eps=eps)
    assert e.value.code == 1 and "eps" in e.value.message
    M.block_norm_dev([p], p, 0, 64, h_out=p, n_out=p, eps=2.0**-126)


def test_a_k_split_is_as_wide_as_the_device_places(rules):
    """No more clusters than run at once, whatever the device's GPCs hold; at least two chunks per CTA."""
    import ctypes as C

    places = [rules.b200, (C.c_uint32 * 9)(132, 132, 132, 128, 112, 264, 264, 256, 224), (C.c_uint32 * 9)(148, 148, 146, 120, 96, 296, 292, 240, 192),
              (C.c_uint32 * 9)(16, 16, 16, 0, 0, 32, 32, 0, 0)]
    for place in places:
        for per_sm in (1, 2):
            room = place[1 + 4 * (per_sm - 1):5 + 4 * (per_sm - 1)]
            for ctas in (1, 2, 7, 16, 32, 33, 60, 66, 74, 100, 148, 149, 300, 5000):
                for chunks in (1, 2, 3, 4, 7, 8, 16, 100):
                    s = rules.log_split(2, chunks, place, ctas, per_sm)
                    fits = [(ctas << i) <= room[i] and chunks >> i >= 2 for i in (1, 2, 3)]
                    assert s == next((i for i, ok in enumerate(fits) if not ok), 3), (list(place), per_sm, ctas, chunks)
    assert rules.log_split(2, 16, places[0], 16, 1) == 2 and rules.log_split(2, 16, places[0], 15, 1) == 3      # fifteen clusters of eight


def test_no_rows_of_empty_tensors_are_no_work():
    """A rank without tokens has empty tensors, whose address is 0; a missing argument is refused as with rows."""
    import torch

    import mimo26f_afd_b200 as M

    e = torch.empty(0, 64)
    assert e.data_ptr() == 0
    w = torch.ones(64)
    M.block_norm_dev([e], e, 0, 64, h_out=e, n_out=e)
    M.block_norm_dev([e, e, e], e, 0, 64, post_w=w, gate=torch.empty(0), gate_kind=M.GATE_TOKEN, pre_w=w, h_out=e, n_out=e)
    M.block_norm_dev([e], None, 0, 64, gate=e, gate_kind=M.GATE_ELEMENT, n_out=e)
    M.block_norm_dev([], e, 0, 64, n_out=e)
    for kw in (dict(residual=None, planes=[]), dict(h_out=None, n_out=None), dict(gate_kind=M.GATE_TOKEN), dict(planes=[e, None]), dict(width=0)):
        a = dict(planes=[e], residual=e, rows=0, width=64, h_out=e, n_out=e)
        a.update(kw)
        with pytest.raises(M.ExpertError) as err:
            M.block_norm_dev(a.pop("planes"), a.pop("residual"), a.pop("rows"), a.pop("width"), **a)
        assert err.value.code == 1


# Requests that CTA pairs run, and the token tile they run with: (BF16, gated, n, k, tokens, tile). Tiles of up to 128 tokens have one scale block
# per piece, wider ones two.
PAIR_SHAPES = [
    (True, False, 305, 4320, 2354, 64), (True, False, 268, 6688, 3645, 112), (True, False, 13250, 1312, 451, 128), (True, False, 9928, 1056, 143, 144),
    (True, False, 10709, 4064, 182, 192), (True, False, 1549, 32, 4038, 224), (True, True, 129, 4544, 2324, 64), (True, True, 14964, 416, 238, 128),
    (True, True, 4867, 1088, 141, 144), (True, True, 5621, 4192, 178, 192), (True, True, 14241, 32, 132, 224),
    (False, False, 260, 6720, 2364, 64), (False, False, 3659, 3008, 1070, 128), (False, False, 564, 2528, 3139, 144), (False, False, 9579, 3808, 145, 160),
    (False, False, 14409, 128, 395, 256), (False, True, 139, 5440, 2346, 64), (False, True, 519, 3104, 3615, 128), (False, True, 4847, 2496, 134, 144),
    (False, True, 14549, 32, 137, 256),
]


def image_tiles(n, gated):
    """128-row tiles of a weight image: an even number; 64 features each when gated, 128 otherwise."""
    return -(-n // (128 if gated else 256)) * 2


def test_the_pair_shapes_run_on_pairs(rules):
    for bf16, gated, n, k, rows, tile in PAIR_SHAPES:
        assert rules.pair_tile(image_tiles(n, gated), -(-k // 128), rules.b200, 148, int(bf16), rows) == tile
    assert {t <= 128 for *_, t in PAIR_SHAPES} == {True, False} and {t for *_, t in PAIR_SHAPES} >= {64, 224, 256}
