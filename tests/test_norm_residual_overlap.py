"""norm_gate_residual and its gradient refuse outputs that overlap each other or an input whose place they cannot take, on
the host: no kernel is launched.  The addresses are never read."""
import pytest

from test_fused_operator_refusals import BF16, norm, norm_backward, refused

ROWS, COLS = 8, 64
T, V = ROWS * COLS * 2, COLS * 2  # bytes of a tensor and of a vector
A = {k: 2 ** 20 * (i + 1) for i, k in enumerate(("h", "x", "w_post", "gate", "w_pre", "x_out", "y"))}
B = {k: 2 ** 20 * (i + 1) for i, k in enumerate(("h", "x", "w_post", "gate", "w_pre", "dx_out", "dy", "dh", "dx", "dw_post", "dgate",
                                                 "dw_pre"))}


@pytest.mark.parametrize("change", [
    {"y": A["x_out"]}, {"y": A["x_out"] + T - 16}, {"x_out": A["h"], "y": A["h"]}, {"x_out": A["h"] + 16}, {"x_out": A["x"] - 16},
    {"y": A["x"] + V}, {"y": A["h"] - T + 2}, {"x_out": A["w_post"]}, {"x_out": A["w_pre"] - T + 16}, {"y": A["gate"]},
    {"group": 4, "x_out": A["gate"] + V},
])
def test_forward(change):
    assert "overlap" in refused(*norm(BF16, rows=ROWS, cols=COLS, **{**A, **change}))


@pytest.mark.parametrize("change", [
    {"dh": B["dx"]}, {"dh": B["dx"] + V}, {"dh": B["h"] + V}, {"dh": B["dy"] - V}, {"dx": B["x"] + V}, {"dx": B["dx_out"] - V},
    {"dx": B["w_post"]}, {"dh": B["gate"]}, {"dw_post": B["dw_pre"]}, {"dw_post": B["dgate"]}, {"dgate": B["dw_pre"] + 2},
    {"dw_pre": B["dh"] + V}, {"dgate": B["dx"]}, {"dgate": B["h"]}, {"dgate": B["w_post"]}, {"group": 4, "dgate": B["gate"] + V},
    {"group": 4, "dw_post": B["dgate"] + V}, {"dh": B["h"], "dx": B["h"]},
])
def test_backward(change):
    assert "overlap" in refused(*norm_backward(BF16, rows=ROWS, cols=COLS, **{**B, **change}))
