"""The language-model training operators through the C++ host layer (argument checks,
shapes, autodiff) on CPU, over the host-memory double of the C ABI, against 64-bit numpy;
and the C ABI's own refusals, which need no GPU."""
import ctypes as C
import importlib.util
import pathlib
import sys

import numpy as np
import pytest

import learn_cases

HERE = pathlib.Path(__file__).resolve().parent


@pytest.fixture(scope="module")
def F():
    sys.path.insert(0, str(HERE / "hostfake"))
    import build_fake

    spec = importlib.util.spec_from_file_location("hostfake.fusion", build_fake.build())
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    return mod


@pytest.mark.parametrize("case", learn_cases.API_CASES, ids=lambda c: c.__name__)
def test_host_layer(F, case):
    case(F)


def test_refusals(F):
    learn_cases.refusals(F)


P = C.c_void_p(4096)  # never read: every call below is refused before a launch

# (function, arguments, what the message names)
BAD_CALLS = [
    ("fz_group_norm", [P, None, None, P, None, None, 1, 1, 6, 4, 1e-5, 0, None, 0, None], "multiple of groups"),
    ("fz_group_norm", [P, None, None, P, None, None, -1, 1, 4, 2, 1e-5, 0, None, 0, None], "negative"),
    ("fz_group_norm", [P, None, None, P, None, None, 1, 1, 4, 2, 1e-5, 9, None, 0, None], "activation"),
    ("fz_group_norm", [P, None, None, P, None, None, 1, 1, 4, 2, -1.0, 0, None, 0, None], "eps"),
    ("fz_group_norm", [P, P, None, P, None, None, 1, 1, 4, 2, 1e-5, 0, None, 0, None], "mean and rstd"),
    ("fz_group_norm", [P, None, None, P, None, None, 1, 1, 4, 2, 1e-5, 0, None, 0, None], "overlap"),
    ("fz_group_norm", [None, None, None, P, None, None, 1, 1, 4, 2, 1e-5, 0, None, 0, None], "null"),
    ("fz_group_norm", [P, None, None, P, None, None, 1 << 40, 1 << 40, 4, 2, 1e-5, 0, None, 0, None], "too many"),
    ("fz_group_norm", [P, None, None, P, None, None, (1 << 30) + 1, 1, 4, 2, 1e-5, 0, None, 0, None], "too many"),
    ("fz_group_norm", [C.c_void_p(8192), None, None, P, None, None, 1, 1 << 24, 8, 2, 1e-5, 0, None, 0, None], "workspace"),
    ("fz_group_norm_backward", [C.c_void_p(8192), P, P, C.c_void_p(12288), P, P, P, None, None, 4, 1, 4, 2, 0, P, 3, None], "workspace"),
    ("fz_group_norm_backward", [P, None, None, None, P, P, P, None, None, 1, 1, 4, 2, 0, None, 0, None], "null"),
    ("fz_group_norm_backward", [P, None, None, P, P, P, P, None, None, 1, 1, 4, 2, 0, None, 0, None], "overlap"),
    ("fz_route", [P, P, P, 4, 1025, 2, 1, None], "FZ_MAX_EXPERTS"),
    ("fz_route", [P, P, P, 4, 8, 9, 1, None], "k must"),
    ("fz_route", [P, P, P, 4, 64, 33, 1, None], "k must"),
    ("fz_route", [P, None, P, 4, 8, 2, 1, None], "null"),
    ("fz_route", [P, P, P, 1 << 31, 8, 2, 1, None], "2^31"),
    ("fz_route_backward", [P, P, P, P, None, 4, 8, 2, 1, None], "null"),
    ("fz_expert_sort", [P, P, P, P, P, 4, 2, 1025, 0, None], "FZ_MAX_EXPERTS"),
    ("fz_expert_sort", [P, P, P, P, P, 4, 2, 8, -1, None], "negative"),
    ("fz_expert_sort", [P, P, P, P, P, 1 << 30, 2, 8, 0, None], "2^31"),
    ("fz_expert_sort", [P, P, P, P, P, 4, 2, 8, 1 << 28, None], "2^31"),
    ("fz_expert_sort", [P, P, None, P, P, 4, 2, 8, 0, None], "null"),
    ("fz_expert_sort", [None, P, P, P, P, 4, 2, 8, 0, None], "null"),
    ("fz_expert_dispatch", [P, None, P, P, 4, 2, 8, 16, None], "null"),
    ("fz_expert_dispatch", [P, P, P, P, 4, 0, 8, 16, None], "k < 1"),
    ("fz_expert_combine", [P, P, P, None, 4, 2, 8, 16, None], "null"),
    ("fz_expert_combine", [P, P, P, P, 4, 2, 1 << 31, 16, None], "2^31"),
    ("fz_expert_combine_backward", [P, P, P, None, P, P, P, 4, 2, 8, 16, None], "null"),
    ("fz_distill", [P, P, P, 7, P, P, None, 2, 8, 3, 1.0, None], "pitch"),
    ("fz_distill", [P, P, P, 8, P, P, None, 2, 8, 1025, 1.0, None], "FZ_MAX_TEACHER"),
    ("fz_distill", [P, P, P, 1 << 24, P, P, None, 2, 1 << 24, 3, 1.0, None], "2^23"),
    ("fz_distill", [P, P, P, 8, P, P, None, 2, 8, 3, 0.0, None], "temperature"),
    ("fz_distill", [P, P, P, 8, P, P, None, 2, 8, 3, float("nan"), None], "temperature"),
    ("fz_distill", [P, None, P, 8, P, P, None, 2, 8, 3, 1.0, None], "null"),
    ("fz_distill_backward", [P, 8, P, P, P, 8, P, P, None, 2, 8, 3, 1.0, None], "overlap"),
    ("fz_distill_backward", [P, 7, P, P, P, 8, P, P, None, 2, 8, 3, 1.0, None], "pitch"),
]


@pytest.mark.parametrize("name,args,says", BAD_CALLS, ids=[f"{i}-{c[0]}-{c[2]}" for i, c in enumerate(BAD_CALLS)])
def test_c_abi_refuses(name, args, says):
    from nova_b200 import capi

    lib = capi.lib()
    assert getattr(lib, name)(*args) == 1  # FZ_ERR_INVALID
    assert says in lib.fz_last_error().decode()


@pytest.mark.parametrize("tau", [-1.0, 9e-19, 1.1e18, 1.9e19, 3e38, float("inf")])
def test_distill_refuses_temperatures_without_a_square(F, tau):
    """The loss's factor tau^2 has to be a normal number: outside [1e-18, 1e18] both directions and
    the module refuse, at the ends they go on to their other checks."""
    from nova_b200 import capi

    lib = capi.lib()
    for name, args in (("fz_distill", lambda t: [P, None, P, 8, P, P, None, 2, 8, 3, t, None]),
                       ("fz_distill_backward", lambda t: [P, 8, P, None, P, 8, P, P, None, 2, 8, 3, t, None])):
        assert getattr(lib, name)(*args(tau)) == 1
        assert "temperature must be in [1e-18, 1e18]" in lib.fz_last_error().decode()
        for end in (1e-18, 1e18):
            assert getattr(lib, name)(*args(end)) == 1 and "null" in lib.fz_last_error().decode()
    T = learn_cases.T
    with pytest.raises(ValueError, match="temperature"):
        F.distill(T(F, np.ones((4, 6))), F.Indices(np.zeros((4, 2), np.int64)), T(F, np.ones((4, 2))), temperature=tau)


def test_empty_calls_launch_nothing():
    """No tokens, rows or elements: nothing to do, and no pointers needed."""
    from nova_b200 import capi

    lib = capi.lib()
    n = lib.fz_launch_count()
    calls = [lib.fz_group_norm(None, None, None, None, None, None, 0, 5, 4, 2, 1e-5, 0, None, 0, None),
             lib.fz_group_norm(None, None, None, None, None, None, 3, 0, 4, 2, 1e-5, 0, None, 0, None),
             lib.fz_route(None, None, None, 0, 8, 2, 1, None),
             lib.fz_route_backward(None, None, None, None, None, 0, 8, 2, 0, None),
             lib.fz_expert_dispatch(None, None, None, None, 0, 2, 0, 16, None),
             lib.fz_expert_combine(None, None, None, None, 0, 2, 0, 16, None),
             lib.fz_expert_combine_backward(None, None, None, None, None, None, None, 0, 2, 0, 16, None),
             lib.fz_distill(None, None, None, 8, None, None, None, 0, 8, 3, 1.0, None),
             lib.fz_distill_backward(None, 8, None, None, None, 8, None, None, None, 0, 8, 3, 1.0, None)]
    assert calls == [0] * len(calls)
    assert lib.fz_launch_count() == n
