"""CPU: where a stage takes the one-launch MoE layer (``fused_moe``)."""

import pytest


@pytest.mark.parametrize("H,F,E,k,rows,fused", [
    (2048, 768, 128, 8, 16, True), (1040, 272, 20, 3, 16, True), (2048, 768, 16, 4, 16, True),
    (2048, 768, 32, 8, 12, True), (2048, 768, 32, 8, 16, False), (4096, 4096, 8, 2, 8, True),
    (4096, 4096, 8, 2, 12, False), (4096, 4096, 8, 4, 12, False), (4096, 2048, 8, 2, 10, True),
    (4096, 2048, 8, 2, 14, False), (256, 128, 16, 4, 16, True),
])
def test_the_faster_form_on_both_sides(H, F, E, k, rows, fused):
    from superl8_serve_b200.runtime import fused_moe_pays

    assert fused_moe_pays(rows, H, F, E, k) == fused
