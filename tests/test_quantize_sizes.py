"""Widths and strides of mt_quantize_f8 at the ends of their ranges, without a GPU."""
import pytest

import mingtts as mt

FAR = 1 << 44  # never dereferenced: every call here is refused


@pytest.mark.parametrize("K,lds,needle", [
    ((1 << 32) - 16, 0, "2^31"),               # 4 ceil(K / 512) of such a K is 0 in 32 bits
    ((1 << 32) - 16, 4, "2^31"),
    ((1 << 31) + 16, (1 << 24) + 4, "2^31"),
    (1 << 31, 1 << 23, "lds"),
    (16, (1 << 24) + 4, "2^24"),
    (16, 1 << 26, "2^24"),                     # 128 values a block: 2^33
])
@pytest.mark.parametrize("norm", [None, FAR // 2])
def test_refused(K, lds, needle, norm):
    if norm and K > 1 << 19:
        needle = "a norm over K"
    rc = mt.load().mt_quantize_f8(FAR, mt.F16, 1, K, K, norm, mt.F16, 1e-6, 2 * FAR, K, 3 * FAR, lds, None)
    assert rc == mt.EINVAL and needle in mt.last_error(), mt.last_error()
