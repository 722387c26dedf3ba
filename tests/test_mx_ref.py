"""The reference of the microscaled formats against values worked by hand."""
import numpy as np

import mx_ref as ref


def _block(*head):
    x = np.zeros((1, 32))
    x[0, :len(head)] = head
    return x


def test_mx4_codes_of_a_block_with_every_tie():
    # largest 6 -> 2^2, scale 2^0: the middles go to the even code, both signs
    c, s = ref.mx4_quantize(_block(6, .25, .75, 1.25, 1.75, 2.5, 3.5, 5, -.25, -.75, -5, -0.0))
    assert s.tolist() == [[127, 0, 0, 0]]
    assert c[0, :6].tolist() == [0x07, 0x22, 0x44, 0x66, 0xA8, 0x8E]
    assert not c[0, 6:].any()


def test_mx4_saturates_and_scales_follow_the_largest_magnitude():
    c, s = ref.mx4_quantize(_block(7.99, -4, 3))        # 2^2 again: 7.99 -> 6
    assert s[0, 0] == 127 and c[0, :2].tolist() == [0xE7, 0x05]
    c, s = ref.mx4_quantize(_block(8, -4, 3))           # 2^3: scale 2: 8 = 4 * 2, -4 = -2 * 2, 3 = 1.5 * 2
    assert s[0, 0] == 128 and c[0, :2].tolist() == [0xC6, 0x03]
    assert ref.mx4_decode(c, s, 3).tolist() == [[8, -4, 3]]


def test_act8_codes():
    c, s = ref.act8_quantize(_block(100, -63.5, 62.5, .5, 1.5))  # 2^6: scale 1, ties to even
    assert s[0, 0] == 127 and c[0, :5].tolist() == [100, -64, 62, 0, 2]
    c, s = ref.act8_quantize(_block(127.9, -127.9))              # would round to 128
    assert c[0, :2].tolist() == [127, -127]
    assert ref.act8_decode(c, s, 2).tolist() == [[127, -127]]


def test_zero_subnormal_and_non_finite_blocks():
    for q in (ref.mx4_quantize, ref.act8_quantize):
        c, s = q(np.zeros((2, 5)))
        assert not s.any() and not c.any()
        c, s = q(_block(2.0 ** -140))
        assert s[0, 0] == 0
        for bad in (np.inf, -np.inf, np.nan):
            c, s = q(_block(1, bad))
            assert s[0, 0] == 255 and not c.any()
    assert np.isnan(ref.mx4_decode(*ref.mx4_quantize(_block(1, np.nan)), 32)).all()
