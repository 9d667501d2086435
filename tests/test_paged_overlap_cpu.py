"""Outputs that share memory with inputs, refused before any device call: queries are rotated, or attended,
in place or apart from what is read."""
import pytest

import lnship
from test_paged_refusals_cpu import EINVAL, P, attn, paged, store

SOUND = (-2, -3)     # as far as the device: LNSHIP_EDEVICE, LNSHIP_ENOINIT


@pytest.fixture(autouse=True)
def no_device():
    import torch
    if torch.cuda.is_available():
        pytest.skip("the pointers here are not device memory")


# 3 rows of 8 heads of 64 are read at P, 512 floats each
@pytest.mark.parametrize("ld,at,out_ld,ok", [
    (512, 0, 512, True),                                      # in place
    (512, 0, 513, False), (513, 0, 512, False),               # the same start, other rows
    (512, 4, 512, False), (512, -4, 512, False), (512, 4 * 511, 512, False), (512, 4 * 512, 512, False),
    (512, 4 * 3 * 512, 512, True), (512, 4 * 3 * 512 - 4, 512, False), (512, -4 * 3 * 512, 512, True),
    (512, -4 * 3 * 512 + 4, 512, False),
    (1024, 4 * 512, 1024, True), (1024, -4 * 512, 1024, True),                # in the gaps
    (1024, 4 * 511, 1024, False), (1024, 4 * 513, 1024, False), (1024, 4 * (512 + 1024), 1024, True),
    (1023, 4 * 512, 1023, False), (1025, 4 * 513, 1025, True), (1024, 4 * 512, 1025, False),
    (600, 4 * (2 * 600 + 512), 700, True), (600, 4 * (2 * 600 + 511), 700, False),
])
def test_outputs_are_the_inputs_or_apart(ld, at, out_ld, ok):
    base = P + (1 << 16)
    want = SOUND if ok else (EINVAL,)
    kv = 1 << 30
    assert store(q=base, q_ld=ld, q_dst=base + at, q_dst_ld=out_ld, k=kv, v=kv) in want
    assert attn(q=base, q_ld=ld, dst=base + at, dst_ld=out_ld) in want


def test_one_row_has_no_stride():
    for a, b in ((512, 777), (777, 512)):
        assert store(paged(ntok=1), q_ld=a, q_dst_ld=b) in SOUND and attn(paged(ntok=1), q_ld=a, dst_ld=b) in SOUND
        assert attn(paged(ntok=1), q_ld=a, dst=P + 4 * 512, dst_ld=b) in SOUND
        assert attn(paged(ntok=1), q_ld=a, dst=P + 4 * 511, dst_ld=b) == EINVAL


def test_rows_in_each_others_gaps():
    import lnship.paged
    apart = lnship.paged._apart
    assert apart(0, 96, 64, 256, 96, 16, 5) and apart(0, 96, 64, 320, 96, 16, 5)      # q, k and v of fused rows
    assert not apart(0, 96, 64, 252, 96, 16, 5) and not apart(0, 96, 64, 324, 96, 16, 5)
    assert not apart(256, 96, 16, 252, 96, 16, 5) and apart(256, 96, 16, 320, 96, 16, 5)
    assert apart(0, 64, 64, 4 * 64 * 5, 64, 64, 5) and not apart(0, 64, 64, 4 * 64 * 5 - 4, 64, 64, 5)
    assert not apart(0, 96, 64, 256, 97, 16, 5) and apart(0, 96, 64, 256, 97, 16, 1)
