"""Workspaces that lie on an operand: refused by pure host logic, no kernel is launched."""
import ctypes as C

import pytest

from composable_kernel_amd import capi

P = 1 << 24


@pytest.mark.parametrize("on", range(8))
@pytest.mark.parametrize("end", ["first", "last"])
def test_a_workspace_of_the_router_on_an_operand(on, end):
    """Ids and counts are indices of the router's second launch: whatever else the workspace holds may not lie there."""
    T, E, k = 5000, 16, 2
    L, d = capi.lib(), capi.RouteDesc(T, E, k, E, 1, 1, 1, capi.SCORE_SOFTMAX, 1, capi.TYPE_F32, 1.0)
    need = L.ckx_route_experts_workspace_bytes(C.byref(d))
    assert need > 0
    ptrs = [P * (i + 1) for i in range(8)]           # logits, bias, number, ids, weights, offsets, rows, places
    size = (T * E * 4, E * 4, 4, T * k * 4, T * k * 4, (E + 1) * 4, T * k * 4, T * k * 4)[on]
    ws = ptrs[on] - need + 16 - need % 16 if end == "first" else ptrs[on] + (size - 1) // 16 * 16
    assert ws % 16 == 0 and ws < ptrs[on] + size and ws + need > ptrs[on]
    assert L.ckx_route_experts(*ptrs, C.byref(d), ws, need, None) == capi.INVALID_VALUE and "the workspace lies on" in capi.last_error()
