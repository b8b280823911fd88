"""Refusals of the expert operations that need no GPU: the options are looked at before the
context is used, and a call of no tokens launches nothing."""
from __future__ import annotations

import ctypes

import pytest

OK, INVALID = 0, 100


def _status(axc, **options):
    lib = axc.load_library()
    nothing = ctypes.create_string_buffer(64)  # stands for a context: a call of no tokens
    o = axc.RouteOptions(**options)._c
    return lib.axh_expert_route(ctypes.addressof(nothing), 0, None, None, None, None, 0,
                                ctypes.byref(o), None)


@pytest.mark.parametrize("n,groups,best,status", [(64, 64, 2, INVALID), (2, 2, 2, INVALID),
                                                  (64, 64, 1, OK), (64, 32, 2, OK), (4, 2, 2, OK),
                                                  (1, 1, 2, OK), (64, 1, 2, OK)])
def test_two_best_of_groups_of_one_expert(axc, n, groups, best, status):
    """Every such group's key would be -inf, and the lowest groups chosen whatever the scores."""
    assert _status(axc, n_experts=n, top_k=1, n_groups=groups, groups_kept=min(groups, 4),
                   group_best=best) == status
