"""Scaled 8-bit pages without a GPU: byte layout, refusals, and the 64-bit restatement the GPU tests compare with."""
import numpy as np
import pytest

from khalamari_b200 import abi, kv_page_write, sliced_kv, sliced_q
from khalamari_b200.device import Dtype
from khalamari_b200.request_page_table import GQAPageTableLayout
from khalamari_b200.sdpa import ExecutionVariant
from khalamari_b200.sdpa import Config as SdpaConfig
from scaled_helpers import CODES, E4M3, make_scaled_case, page_bytes, quantise, reference, values_of

KINDS = {"int8": Dtype.Int8Scaled, "e4m3": Dtype.Fp8E4M3Scaled}
LAYOUT = GQAPageTableLayout(2, 1, 4, 1)


@pytest.mark.parametrize("kind", KINDS.values())
@pytest.mark.parametrize("hkv,d,page", [(1, 128, 8), (8, 128, 16), (2, 256, 32), (5, 256, 16)])
def test_page_bytes_hold_codes_and_scale_bytes(kind, hkv, d, page):
    config = kv_page_write.Config(hkv, d, page_bytes(hkv, page, d), Dtype.Bfloat16, kind)
    assert config.num_tokens_per_page() == page
    kv = sliced_kv.Config(hkv * 2, hkv, d, 0.1, page_bytes(hkv, page, d), LAYOUT, Dtype.Bfloat16, kind)
    assert kv.num_tokens_per_page() == page
    q = sliced_q.Config(hkv * 2, hkv, d, 0.1, page_bytes(hkv, page, d), Dtype.Float16, LAYOUT, kind)
    if (d, page) in ((128, 8), (128, 16), (256, 8), (256, 16), (256, 32)):
        variant = ExecutionVariant.sliced_q(SdpaConfig(Dtype.Float16, hkv * 2, hkv, d, page), 2, 8, 16, 2)
        assert q.sizes(variant, sliced_q.Shape(8, 1, 1)).num_tokens_per_page == page


@pytest.mark.parametrize("kind", KINDS.values())
def test_unsupported_geometries_are_refused(kind):
    with pytest.raises(abi.InvalidArgument, match="head_dim 128 and 256"):
        kv_page_write.Config(2, 64, page_bytes(2, 16, 64), Dtype.Bfloat16, kind).validate()
    with pytest.raises(abi.InvalidArgument, match="8, 16 or 32 tokens"):
        kv_page_write.Config(2, 128, page_bytes(2, 24, 128), Dtype.Bfloat16, kind).validate()
    with pytest.raises(abi.InvalidArgument, match="divisible"):
        kv_page_write.Config(2, 128, 2 * 2 * 16 * 128, Dtype.Bfloat16, kind).validate()  # codes without scale bytes
    with pytest.raises(abi.InvalidArgument, match="at least one token"):
        kv_page_write.Config(2, 128, 0, Dtype.Bfloat16, kind).validate()
    with pytest.raises(abi.InvalidArgument, match="BF16"):
        kv_page_write.Config(2, 128, page_bytes(2, 16, 128), Dtype.Float32, kind).validate()
    with pytest.raises(abi.InvalidArgument, match="must fit u64|must fit u32"):
        kv_page_write.Config(0xFFFFFFFF, 0xFFFFFFFF, 16, Dtype.Bfloat16, kind).validate()


def test_row_bytes():
    assert Dtype.Int8Scaled.kv_row_bytes(128) == Dtype.Fp8E4M3Scaled.kv_row_bytes(128) == 129
    assert Dtype.Fp8E4M3FN.kv_row_bytes(128) == 128 and Dtype.Bfloat16.kv_row_bytes(128) == 256


def test_null_arguments_are_refused():
    with pytest.raises(abi.InvalidArgument, match="null argument"):
        abi.call("kh_kv_page_read_create", None, None, None)
    with pytest.raises(abi.InvalidArgument, match="null argument"):
        abi.call("kh_kv_page_read_invoke", None, None, None, None, 1, 0)
    abi.call("kh_kv_page_read_destroy", None)


@pytest.mark.parametrize("code", CODES)
def test_restated_rows_are_within_half_a_step(code):
    rng = np.random.default_rng(5)
    rows = rng.standard_normal((300, 128)) * np.exp2(rng.integers(-60, 60, (300, 1)))
    rows[7] = 0.0
    codes, scale = quantise(rows, code)
    back = values_of(codes, scale, code)
    top = np.abs(rows).max(-1, keepdims=True)
    power = np.exp2(scale.astype(float) - 127)[:, None]
    assert scale[7] == 0 and not back[7].any()
    if code == "int8":
        half = 0.5 * power
        assert np.all(np.abs(codes.astype(np.int8).astype(int)) <= 127)
    else:  # half a step of the code: 2^-4 of the value, or 2^-10 of the scale among the subnormals
        half = np.maximum(np.abs(rows) * 2.0 ** -4, 2.0 ** -10 * power)
        assert np.all(np.isfinite(E4M3[codes]))
    assert np.all(np.abs(back - rows) <= half * (top > 0))
    # the scale is the smallest that fits
    keep = np.delete(np.arange(300), 7)
    smaller = top[keep, 0] / (power[keep, 0] / 2)
    assert np.all(np.rint(smaller) > 127) if code == "int8" else np.all(smaller > 448)


@pytest.mark.parametrize("code", CODES)
def test_restated_attention_matches_a_softmax_over_the_decoded_rows(code):
    case = make_scaled_case(1, code, "f16", 4, 2, 128, [5, 0], [1, 3])
    out, _ = reference(case)
    q = case.q_bits.view(np.float16).astype(float).reshape(-1, 4, 128)
    k, v = case.k[1][:2, 1], case.v[1][:2, 1]
    w = np.exp(k @ q[2, 3] * case.scale)
    assert np.allclose(out[2, 3], w @ v / w.sum(), rtol=1e-12, atol=1e-12)


@pytest.mark.parametrize("hq,hkv,d,q_len,history,whole", [
    (64, 8, 128, 2048, 3900, True),    # 1,024 tasks
    (64, 8, 128, 256, 3900, False),    # 128 tasks: fewer than SMs
    (16, 2, 256, 2048, 3900, False),   # 256 tasks, one tile at a time
    (32, 4, 256, 2048, 3900, True),    # 512 tasks
])
def test_the_chained_policy_keeps_wide_tiles_whole_from_fewer_tasks_on(hq, hkv, d, q_len, history, whole):
    from khalamari_b200.replay import GQAReplayBucketPolicy
    from khalamari_b200.selector import RequestShape, Selector, SelectorPolicy
    layout = GQAPageTableLayout(1, 1, 1024, 1)
    for policy, expected in ((SelectorPolicy.B200Chained, whole), (SelectorPolicy.B200, False)):
        selector = Selector.for_lookup(SdpaConfig(Dtype.Bfloat16, hq, hkv, d, 16), 4096, layout)
        selector.set_policy(policy, 148)
        limits = selector.limits()
        buckets = GQAReplayBucketPolicy(limits.max_tokens, limits.max_map_task_templates)
        selection = selector.select([RequestShape(history, q_len)], buckets, q_len)
        assert selection.direct_output() == expected
