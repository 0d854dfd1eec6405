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
