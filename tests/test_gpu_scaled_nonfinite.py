"""Q rows that are not finite over scaled 8-bit pages (``-m gpu``): every score of such a row is an infinity or NaN, so its
softmax is NaN, on whatever route the batch takes, and no other row is touched."""
import numpy as np
import pytest

from helpers import round_to
from scaled_helpers import CODES, ScaledRun, assert_close, make_scaled_case, planes, quantise, reference, values_of

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def device():
    from khalamari_b200.device import Device
    return Device(0)


SHAPES = [
    # hq, hkv, d, histories, q_lens
    (16, 2, 128, [1999, 40, 333], [1, 1, 1]),     # one token each
    (12, 1, 128, [1999, 40], [1, 1]),
    (16, 2, 256, [1999, 40, 333], [1, 1, 1]),
    (24, 2, 256, [900, 40], [1, 1]),
    (24, 4, 256, [700, 61], [4, 4]),              # verify
    (24, 4, 128, [700, 61], [4, 3]),
    (16, 2, 128, [900, 0], [150, 40]),            # wide tiles, cut
    (16, 2, 256, [900, 0], [50, 40]),
    (16, 2, 128, [0], [200]),                     # wide tiles, direct output
    (16, 2, 256, [0], [200]),
]


@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("io", ["bf16", "f16"])
@pytest.mark.parametrize("sign", [1, -1])
@pytest.mark.parametrize("hq,hkv,d,histories,q_lens", SHAPES)
def test_an_infinity_in_q_makes_its_row_nan(device, code, io, sign, hq, hkv, d, histories, q_lens):
    """One element of K is positive in all tokens, and Q holds an infinity there: all scores of the row are +inf or all -inf."""
    case = make_scaled_case(hq + d + q_lens[0], code, io, hq, hkv, d, histories, q_lens)
    codes, scales = planes(case.pool, hkv, 16, d)
    for r, context in enumerate(h + n for h, n in zip(histories, q_lens)):
        k = case.k[r].copy()
        k[:, :, 5] = np.abs(k).max(-1)  # (the row's largest code, so that its scale stays)
        case.k[r] = values_of(*quantise(k, code), code)
        t = np.arange(context)
        codes[case.table[case.slots[r], 0, t // 16], 0, :, t % 16], scales[case.table[case.slots[r], 0, t // 16], :, 0, t % 16] = quantise(k, code)
    infinity, _ = round_to(io, np.array([sign * np.inf], np.float32))
    q = case.q_bits.reshape(-1, hq, d)
    hidden = np.zeros(q.shape[:2], bool)
    for token, head in ((0, 1), (len(q) - 1, hq - 1), (len(q) // 2, 0)):
        hidden[token, head] = True
    plain = case.q_bits.copy()
    q[hidden, 5] = infinity[0]
    run = ScaledRun(device, case, max_tokens=256)
    run.plan()
    run.record()
    out = run.read()
    assert np.isnan(out[hidden]).all()
    case.q_bits = plain
    expected, bound = reference(case, wide=run.wide())
    assert_close(out[~hidden], expected[~hidden], bound[~hidden])
