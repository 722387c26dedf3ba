"""What the host side of the microscaled operators decides before a launch, seen through the workspaces it asks for and
the calls it refuses.  No kernel is launched here."""
import pytest

from necklace_amd import _lib

TYPES = range(3)


@pytest.mark.parametrize("ty", TYPES)
def test_a_bias_gradient_alone_is_cut_as_its_workgroups_need(ty):
    """k = 0: a workgroup for 64 lanes of 16 bytes of a row; parts only until there are two for each of 256 CUs."""
    need = _lib.mx_lib().nkmx_act8_wgrad_workspace
    width = 256 if ty == 0 else 512
    for n in (width * 512, 1 << 20):
        assert need(ty, 16384, n, 0) == 0
    for t, n in ((16384, 4096), (16384, 20000), (200000, 640), (5000, 30000), (2 ** 31 - 1, 64)):
        assert need(ty, t, n, 0) <= min(64, 512 // -(-n // width)) * (n + 3) * 4
    assert need(ty, 64, 64, 0) == 0


FAR = 1 << 40


def test_an_activation_without_its_checkpoint_is_named_by_two_null_pointers():
    save = _lib.mx_lib().nkmx_act8_save
    assert save(FAR, 2 * FAR, 0, 1, 0, 300, 300, 300, None, None, None) == 0
    # past the check of the codes: y overlaps x
    assert save(FAR, FAR + 4, 0, 1, 4, 300, 300, 300, None, None, None) == -4
    assert save(FAR, 2 * FAR, 0, 1, 4, 300, 300, 300, 3 * FAR, None, None) == -1
    assert save(FAR, 2 * FAR, 0, 1, 4, 300, 300, 300, None, 3 * FAR, None) == -1
    assert save(FAR, None, 0, 0, 4, 300, 300, 300, None, None, None) == -1  # no activation: nothing to do but save


def test_launches_of_too_many_threads_are_refused():
    """Sizes below 2^31 whose launch would take 2^32 threads: an argument error, before anything reaches a GPU."""
    L, big = _lib.mx_lib(), 2 ** 31 - 1
    matmul = lambda m, n, k: L.nkmx_mx4_matmul(FAR, 1, m, n, k, n, 2 * FAR, 3 * FAR, 4 * FAR, 5 * FAR, None, None)  # noqa: E731
    assert matmul(1, big, 64) == -3 and matmul(16, 2 ** 28, 64) == -3 and matmul(big, 64, 64) == -3 and matmul(big, 1, 0) == -3
    assert L.nkmx_mx4_quantize(FAR, 0, 1, big, big, 2 * FAR, 3 * FAR, 1, None) == -3
    assert L.nkmx_mx4_linear(FAR, 2 * FAR, 1, 1, big, 1, big, 1, 3 * FAR, 4 * FAR, None, 5 * FAR, 1 << 20, None) == -3
    for ty in TYPES:
        assert L.nkmx_act8_wgrad(FAR, None, 2 * FAR, ty, 1, big, 1, 1, big, 3 * FAR, 4 * FAR, 0, None, 0, None) == -3
