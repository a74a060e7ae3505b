"""CPU: sizes that the router's grid cannot hold are argument errors, not launch failures."""

from primus_turbo_b200 import _lib


def test_tokens_past_the_grid_are_refused():
    L, p, f32 = _lib.lib, 0x1000, _lib.PTB_F32
    most = 4 * (2**31 - 1)  # four tokens a CTA
    for T in (most + 1, 2 * most):
        assert L.ptb_topk_router(p, f32, T, 8, 8, 2, 0, None, 1, 1, 0, 1.0, p, p, None, None, None) == -5
        assert L.ptb_topk_router_bwd(p, f32, T, 8, 8, 2, 0, 0, 1.0, p, p, 2, 0, p, None) == -5
