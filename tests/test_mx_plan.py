"""What the host side of the microscaled operators decides before a launch, seen through the workspaces it asks for and
the calls it refuses.  No kernel is launched here."""
import pytest

from necklace_amd import _lib

TYPES = range(3)


@pytest.mark.parametrize("ty", TYPES)
def test_a_bias_gradient_alone_is_cut_as_its_workgroups_need(ty):
    """k = 0: one workgroup for 64 columns of dy; parts only until they fill the chip (256 CUs, 3 workgroups each)."""
    need = _lib.mx_lib().nkmx_act8_wgrad_workspace
    for n in (65536, 100000, 1 << 20):  # 1024 workgroups and more
        assert need(ty, 16384, n, 0) == 0
    for t, n in ((16384, 4096), (16384, 20000), (200000, 640), (5000, 30000)):
        assert need(ty, t, n, 0) <= 768 // -(-n // 64) * (n + 3) * 4
    assert need(ty, 64, 64, 0) == 0  # a single stage
