"""Arrays that the C entry points of the q/k norm + RoPE cannot do without
(no launch is made: every call here is refused, or has nothing to do)."""
import pytest

from forge_hip import _lib as L

S4 = (16, 0, 0, 0)
NONE = (None, 0, 0, 0)


def _fwd(q=S4, k=S4, qo=S4, ko=S4, weights=(16, 16), tables=(16, 0, 0, 16, 0, 0), sizes=(1, 4, 2, 8, 128)):
    return L.forge_qk_norm_rope_fwd(2, *q, *k, *qo, *ko, *weights, 2, *tables, 2, 8, None, *sizes, 1e-6, 0.0, None)


def _bwd(dq=S4, dk=S4, q=S4, k=S4, qi=S4, ki=S4, weights=(16, 16), tables=(16, 0, 0, 16, 0, 0), sizes=(1, 4, 2, 8, 128)):
    return L.forge_qk_norm_rope_bwd(2, *dq, *dk, *q, *k, *qi, *ki, *weights, 2, *tables, 2, 8, None, None, None, None,
                                    *sizes, 1e-6, 0.0, None)


@pytest.mark.parametrize("change", [{"q": NONE}, {"k": NONE}, {"qo": NONE}, {"ko": NONE}, {"weights": (None, 16)},
                                    {"weights": (16, None)}, {"tables": (None, 0, 0, 16, 0, 0)},
                                    {"tables": (16, 0, 0, None, 0, 0)}], ids=str)
def test_forward_refuses_null_arrays(change):
    assert _fwd(**change) == 1 and b"NULL" in L.forge_last_error()


@pytest.mark.parametrize("change", [{"dq": NONE}, {"dk": NONE}, {"q": NONE}, {"k": NONE}, {"qi": NONE}, {"ki": NONE},
                                    {"weights": (None, 16)}, {"weights": (16, None)},
                                    {"tables": (None, 0, 0, 16, 0, 0)}], ids=str)
def test_backward_refuses_null_arrays(change):
    assert _bwd(**change) == 1 and b"NULL" in L.forge_last_error()


@pytest.mark.parametrize("sizes", [(0, 4, 2, 8, 128), (1, 4, 2, 0, 128), (1, 0, 0, 8, 128)])
def test_nothing_to_do_needs_no_arrays(sizes):
    no = {"q": NONE, "k": NONE, "weights": (None, None), "tables": (None, 0, 0, None, 0, 0), "sizes": sizes}
    assert _fwd(qo=NONE, ko=NONE, **no) == 0
    assert _bwd(dq=NONE, dk=NONE, qi=NONE, ki=NONE, **no) == 0


def test_a_side_without_heads_needs_no_arrays():
    """n_kv = 0: k's arrays are not looked at (here q's are refused instead)."""
    sizes = (1, 4, 0, 8, 128)
    assert _fwd(q=NONE, k=NONE, ko=NONE, weights=(16, None), sizes=sizes) == 1
    assert b"q or k" in L.forge_last_error()
