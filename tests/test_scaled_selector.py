"""Selections over scaled 8-bit pages, on the host: the slices a batch is cut into go by the kernel that its tiles run on."""
import pytest

from khalamari_b200.device import Dtype
from khalamari_b200.replay import GQAReplayBucketPolicy
from khalamari_b200.request_page_table import GQAPageTableLayout
from khalamari_b200.sdpa import Config as SdpaConfig
from khalamari_b200.selector import RequestShape, Selector, SelectorPolicy


def _select(policy, hq, hkv, d, requests, tokens_per_page=16):
    longest = max(h + n for h, n in requests)
    layout = GQAPageTableLayout(len(requests), 1, -(-longest // tokens_per_page), 1)
    selector = Selector.for_lookup(SdpaConfig(Dtype.Bfloat16, hq, hkv, d, tokens_per_page), 8192, layout)
    selector.set_policy(policy, 148)
    limits = selector.limits()
    buckets = GQAReplayBucketPolicy(limits.max_tokens, limits.max_map_task_templates)
    return selector.select([RequestShape(h, n) for h, n in requests], buckets, sum(n for _, n in requests))


@pytest.mark.parametrize("hq,hkv,d,q_len,merged", [
    (24, 4, 256, 4, True),     # 24 rows: the kernel that merges slices
    (16, 2, 256, 4, False),    # 32 rows at head_dim 256: tensor memory, every slice a partial of its own
    (28, 4, 256, 4, False),    # 28 rows
    (32, 1, 256, 1, False),    # one token, 32 heads
    (64, 8, 128, 4, True),     # 32 rows at head_dim 128
    (12, 2, 128, 8, False),    # 48 rows
])
def test_only_tiles_whose_slices_are_merged_get_finer_slices(hq, hkv, d, q_len, merged):
    requests = [(16000, q_len)] * 32
    plain, chained = (len(_select(p, hq, hkv, d, requests).map_task_templates())
                      for p in (SelectorPolicy.B200, SelectorPolicy.B200Chained))
    assert chained > plain if merged else chained == plain


@pytest.mark.parametrize("hq,hkv,d,requests,whole", [
    (4, 4, 256, [(4000, 2048)] * 2, True),    # 512 tasks of 32 rows at head_dim 256: at least two an SM
    (4, 4, 256, [(4000, 1024)], False),       # 128 tasks
    (4, 4, 128, [(4000, 2048)] * 2, False),   # 32 rows at head_dim 128 are not wide
    (8, 4, 128, [(4000, 2048)] * 2, True),
])
def test_wide_tiles_stay_whole_from_the_same_width_on(hq, hkv, d, requests, whole):
    assert _select(SelectorPolicy.B200Chained, hq, hkv, d, requests).direct_output() == whole
