"""Blocks whose largest value is below the floor of 1e-10: the divisor is then a float32 of 24 significant bits, and the argument that rounds the
product with 448 / amax to multiples of 8 units rests on 11.  For bf16 (fp16 has no such values) it is checked for every magnitude."""

import numpy as np


def test_codes_of_every_bf16_magnitude_below_the_floor():
    floor = np.float32(1e-10)
    assert floor.view(np.uint32) == 0x2EDBE6FF
    bits = np.arange(0, 0x7F80, dtype=np.uint32) << 16
    x = bits.view(np.float32)
    x = x[x < floor]
    assert x.size == 11996
    product = x * (np.float32(448) / floor)
    kernel = ((product.view(np.uint32) + np.uint32(4)) & np.uint32(0xFFFFFFF8)).view(np.float32)

    def e4m3(v):
        v = v.astype(np.float64)
        step = np.exp2(np.maximum(np.frexp(v)[1] - 1, -6) - 3)
        return np.rint(v / step) * step

    assert (e4m3(kernel) == e4m3(x.astype(np.float64) * 448 / np.float64(floor))).all()
