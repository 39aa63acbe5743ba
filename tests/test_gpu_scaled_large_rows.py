"""Scaled 8-bit pages and cached rows at the top of their type's range (``-m gpu``): a row of the type's largest value stands
for one step more (2^128 from bf16, 2^16 from f16), which must not turn into infinities or NaN on the way."""
import numpy as np
import pytest

from helpers import bits_to_f32, round_to
from scaled_helpers import CODES, ScaledRun, assert_close, make_scaled_case, planes, quantise, reference, values_of

pytestmark = pytest.mark.gpu

MOST = {"bf16": float(np.uint32(0x7F7F0000).view(np.float32)), "f16": 65504.0}


@pytest.fixture(scope="module")
def device():
    from khalamari_b200.device import Device
    return Device(0)


def _put(case, request, tokens, k=None, v=None):
    """Replaces cached rows [len(tokens), Hkv, D] of one request: quantised here, as the page write does."""
    codes, scales = planes(case.pool, case.hkv, case.page, case.d)
    tokens = np.asarray(tokens)
    at, row = case.table[case.slots[request], case.layer, tokens // case.page], tokens % case.page
    for plane, (held, x) in enumerate(((case.k, k), (case.v, v))):
        if x is None:
            continue
        _, x = round_to(case.dtype_name, np.broadcast_to(x, (len(tokens), case.hkv, case.d)).astype(np.float32))
        c, b = quantise(x, case.code)
        codes[at, plane, :, row] = c
        scales[at, :, plane, row] = b
        held[request] = held[request].copy()
        held[request][tokens] = values_of(c, b, case.code)


@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("io", ["bf16", "f16"])
@pytest.mark.parametrize("hq,hkv,d,histories,q_lens", [
    (16, 2, 128, [300], [64]), (16, 2, 256, [300], [64]), (24, 4, 128, [40], [4]), (24, 4, 256, [40], [4]), (8, 8, 128, [0], [24]),
])
def test_a_largest_row_reaches_only_the_queries_that_see_it(device, code, io, hq, hkv, d, histories, q_lens):
    """The new chunk's middle token holds V rows of the largest value: earlier queries share its step and must not see it."""
    case = make_scaled_case(d + hq, code, io, hq, hkv, d, histories, q_lens)
    middle = q_lens[0] // 2 + q_lens[0] // 12
    _put(case, 0, [histories[0] + middle], v=MOST[io])
    run = ScaledRun(device, case, max_tokens=256)
    run.plan()
    run.record()
    out = run.read()
    expected, bound = reference(case, wide=run.wide())
    assert_close(out[:middle], expected[:middle], bound[:middle], "queries before the token")
    assert not np.isnan(out).any()


@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("io", ["bf16", "f16"])
@pytest.mark.parametrize("hq,hkv,d,q_len", [(16, 2, 128, 1), (12, 1, 128, 1), (16, 2, 256, 1), (24, 2, 256, 1), (24, 4, 128, 4),
                                            (24, 4, 256, 4), (16, 2, 128, 64), (16, 2, 256, 64)])
def test_an_average_of_largest_rows_is_the_largest_value(device, code, io, hq, hkv, d, q_len):
    """All V rows alike: the output is that row, as it was before it was quantised."""
    case = make_scaled_case(3, code, io, hq, hkv, d, [0], [q_len])
    signs = np.where(np.arange(d) % 3 == 0, -1.0, 1.0)
    _put(case, 0, np.arange(q_len), v=MOST[io] * signs)
    out = ScaledRun(device, case, max_tokens=256).run()
    if q_len <= 4:
        assert np.array_equal(out, np.broadcast_to(MOST[io] * signs, out.shape).astype(np.float32))
    else:
        # probabilities are rounded on their own (half a step each), the sum is not
        assert np.all(np.abs(out / signs - MOST[io]) <= MOST[io] * 2.02 * (2.0 ** -8 if io == "bf16" else 2.0 ** -11))


@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("hq,hkv,d,batch", [(8, 1, 128, 64), (16, 2, 128, 64), (8, 1, 256, 64), (12, 1, 256, 296)])
def test_scores_that_rise_within_a_factor_before_the_largest_rows(device, code, hq, hkv, d, batch):
    """Every other 16-token tile scores 2^7.5 times higher than the one before it, close to the factor from which running
    references are raised, and V rows reach 2^127.3: no intermediate factor may leave f32."""
    context = 256
    case = make_scaled_case(11, code, "bf16", hq, hkv, d, [context - 1] * batch, [1] * batch)
    rng = np.random.default_rng(12)
    case.q_bits[:] = round_to("bf16", np.ones((1,), np.float32))[0][0]
    # scores: d * a * d^-1/2 in the natural log domain
    a = 7.5 * np.log(2.0) / np.sqrt(d) * ((np.arange(context) // 16) % 2)
    for r in range(batch):
        v = 1.2 * 2.0 ** 127 * rng.choice([-1.0, 1.0], (context, hkv, d))
        _put(case, r, np.arange(context), k=np.broadcast_to(a[:, None, None], (context, hkv, d)), v=v)
    run = ScaledRun(device, case, max_tokens=512)
    variant = next(v for v in run.attention.selector.variants() if v.kind == 0 and v.thread_block.max_q_tokens == 1) \
        if hq // hkv <= 8 else None
    selection = None if variant is None else run.attention.select_partitioned(variant, context, False, case.histories, case.cu)
    out = run.run(selection)
    # one distinct query: the reference of one head a KV head serves the group
    expected, bound = reference(case)
    assert_close(out, expected, bound)


@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("power", [-122, -60, 100])
@pytest.mark.parametrize("hq,hkv,d,histories,q_lens", [
    (16, 2, 128, [300, 33], [1, 1]), (24, 2, 256, [300, 33], [1, 1]), (24, 4, 256, [90], [4]), (16, 2, 128, [300], [64]), (16, 2, 256, [300], [64]),
])
def test_rows_of_q_and_k_whose_sizes_cancel(device, code, power, hq, hkv, d, histories, q_lens):
    """Q of size 2^power against K of size 2^(-1 - power): the scores are ordinary, the operands reach both ends of bf16's range."""
    case = make_scaled_case(17, code, "bf16", hq, hkv, d, histories, q_lens)
    case.q_bits[:] = round_to("bf16", (bits_to_f32("bf16", case.q_bits) * np.float32(2.0 ** power)).astype(np.float32))[0].reshape(case.q_bits.shape)
    for r, k in enumerate(case.k):
        _put(case, r, np.arange(len(k)), k=k * 2.0 ** (-1 - power))
    run = ScaledRun(device, case, max_tokens=256)
    out = run.run()
    assert_close(out, *reference(case, wide=run.wide()))
