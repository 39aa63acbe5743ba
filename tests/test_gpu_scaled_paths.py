"""Scaled 8-bit pages on the framework's other paths (``-m gpu``): 32-token pages at head_dim 128, chains of more slices than a
pass holds, one dominant token, host buffers, and the bidirectional-block composite over a scaled history."""
import numpy as np
import pytest

from helpers import bits_to_f32, round_to
from scaled_helpers import CODES, ScaledRun, assert_close, make_scaled_case, page_bytes, planes, quantise, reference, values_of

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def device():
    from khalamari_b200.device import Device
    return Device(0)


# ---- 32-token pages at head_dim 128: any number of new tokens runs as single-token tasks -------------------------------
@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("io", ["bf16", "f16"])
@pytest.mark.parametrize("hq,hkv,histories,q_lens", [
    (64, 8, [699, 32, 0, 1499], [1, 1, 1, 1]), (12, 1, [30, 31, 63, 95], [1, 1, 1, 1]), (16, 2, [700, 0], [40, 33]), (7, 1, [500], [3]),
])
def test_pages_of_32_tokens_at_head_dim_128(device, code, io, hq, hkv, histories, q_lens):
    case = make_scaled_case(hq + len(q_lens), code, io, hq, hkv, 128, histories, q_lens, page=32, layers=2, layer=1)
    run = ScaledRun(device, case, max_tokens=256)
    out = run.run()
    assert run.attention.metadata.variant().thread_block.max_q_tokens == 1 or not run.wide()
    assert_close(out, *reference(case, wide=run.wide()))


@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("io", ["bf16", "f16"])
def test_pages_of_32_tokens_at_head_dim_128_are_written_and_read(device, code, io):
    from khalamari_b200 import kv_page_read, kv_page_write
    from khalamari_b200.device import Buffer, Dtype, Stream
    from khalamari_b200.request_page_table import GQAPageTableLayout
    rng = np.random.default_rng(5)
    hkv, d, page, pages = 3, 128, 32, 4
    dtype = Dtype.Bfloat16 if io == "bf16" else Dtype.Float16
    kind = Dtype.Int8Scaled if code == "int8" else Dtype.Fp8E4M3Scaled
    n = 3 * page - 5
    (k_bits, k), (v_bits, v) = (round_to(io, rng.standard_normal((n, hkv, d)).astype(np.float32)) for _ in range(2))
    table = np.array([3, 0, 2], np.uint32)
    expected = np.full(pages * page_bytes(hkv, page, d), 0x55, np.uint8)
    codes, scales = planes(expected, hkv, page, d)
    tokens = rng.permutation(3 * page)[:n]
    for plane, x in enumerate((k, v)):
        c, b = quantise(x, code)
        codes[table[tokens // page], plane, :, tokens % page] = c
        scales[table[tokens // page], :, plane, tokens % page] = b
    config = kv_page_write.Config(hkv, d, page_bytes(hkv, page, d), dtype, kind)
    layout, stream = GQAPageTableLayout(1, 1, 3, 1), Stream(device)
    pool = Buffer.from_slice(device, np.full(expected.size, 0x55, np.uint8))
    index = [Buffer.from_slice(device, x) for x in (np.zeros(n, np.uint32), tokens.astype(np.uint32), table)]
    rows = [Buffer.from_slice(device, x) for x in (k_bits, v_bits)]
    kv_page_write.Compute(device, config).invoke(stream, kv_page_write.Shape(n, layout), kv_page_write.Buffers(pool, *rows, *index), n)
    outs = [Buffer.new_zeroed(device, n * hkv * d * 2) for _ in range(2)]
    kv_page_read.Compute(device, config).invoke(stream, kv_page_read.Shape(n, layout), kv_page_read.Buffers(pool, *outs, *index), n)
    stream.synchronize()
    assert device.check(stream) == 0
    assert np.array_equal(pool.read(0, expected.size, np.uint8), expected)
    for out, x in zip(outs, (k, v)):
        got = bits_to_f32(io, out.read(0, n * hkv * d, np.uint16)).reshape(n, hkv, d)
        back = values_of(*quantise(x, code), code)
        # exact in bf16; in f16 a code times 2^e below 2^-14 is rounded to its subnormals
        assert np.array_equal(got, back.astype(np.float32)) if io == "bf16" else np.abs(got - back).max() <= 2.0 ** -25


# ---- long chains ---------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("hq,hkv,d", [(16, 2, 128), (5, 1, 128), (16, 2, 256)])
def test_chains_of_more_slices_than_a_pass_holds(device, code, hq, hkv, d):
    """313 and 130 slices of one sequence: more than the 128 items of a pass, and than the parts a chain may be cut into freely."""
    case = make_scaled_case(9, code, "bf16", hq, hkv, d, [4999, 2079, 64], [1, 1, 1])
    run = ScaledRun(device, case, max_tokens=2048)
    variant = next(v for v in run.attention.selector.variants() if v.kind == 0 and v.thread_block.max_q_tokens == 1)
    selection = run.attention.select_partitioned(variant, 16, False, case.histories, case.cu)
    assert len(selection.map_task_templates()) == 313 + 130 + 5
    assert_close(run.run(selection), *reference(case))


@pytest.mark.parametrize("code", CODES)
def test_long_chains_on_many_sequences(device, code):
    """16 sequences whose slices outnumber a pass: every CTA walks several passes."""
    contexts = [2048 + 97 * i for i in range(16)]
    case = make_scaled_case(10, code, "bf16", 24, 1, 256, [c - 4 for c in contexts[:4]], [4] * 4)
    run = ScaledRun(device, case, max_tokens=4096)
    run.plan()
    chosen = run.attention.metadata.variant()
    selection = run.attention.select_partitioned(chosen, 16, False, case.histories, case.cu)
    out = run.run(selection)
    assert_close(out, *reference(case, wide=run.wide()))
    case = make_scaled_case(10, code, "bf16", 8, 1, 128, [c - 1 for c in contexts], [1] * 16)
    run = ScaledRun(device, case, max_tokens=4096)
    variant = next(v for v in run.attention.selector.variants() if v.kind == 0 and v.thread_block.max_q_tokens == 1)
    assert_close(run.run(run.attention.select_partitioned(variant, 16, False, case.histories, case.cu)), *reference(case))


@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("d,slice_tokens", [(128, 1 << 17), (128, 512), (256, 1 << 17)])
def test_one_dominant_token_of_a_long_sequence(device, code, d, slice_tokens):
    """70,000 tokens whose V rows agree in sign, and one token that outweighs any other 2^17 times: small weights are
    rounded relative to the dominant one in the warp that holds it, in one work item or in 137."""
    context = 70000
    case = make_scaled_case(14, code, "bf16", 8, 1, d, [context - 1], [1], v_scale=lambda rng, n, h: np.full((n, h), 1.0))
    q = bits_to_f32("bf16", case.q_bits)[0, 0].astype(np.float64)
    codes, scales = planes(case.pool, 1, 16, d)
    tokens = np.arange(context)
    at = case.table[case.slots[0], 0, tokens // 16]
    k = case.k[0] * 0.05
    k[31000, 0] = q * (17 * np.log(2.0) / (case.scale * (q @ q)))  # head 0: 17 in the log2 domain
    for plane, x in ((0, k), (1, np.abs(case.v[0]))):
        _, x = round_to("bf16", x.astype(np.float32))
        c, b = quantise(x, code)
        codes[at, plane, :, tokens % 16] = c
        scales[at, :, plane, tokens % 16] = b
        (case.k, case.v)[plane][0] = values_of(c, b, code)
    run = ScaledRun(device, case, max_tokens=2048)
    variant = next(v for v in run.attention.selector.variants() if v.kind == 0 and v.thread_block.max_q_tokens == 1)
    selection = run.attention.select_partitioned(variant, slice_tokens, False, case.histories, case.cu)
    assert_close(run.run(selection), *reference(case))


# ---- host buffers ----------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("code", CODES)
def test_host_steps_over_scaled_pages(device, code):
    """``attend_host`` and two steps in flight give the resident path's bits."""
    from khalamari_b200.device import PinnedArray
    from khalamari_b200.gqa import HostPipeline
    case = make_scaled_case(64, code, "bf16", 64, 8, 128, [1499, 699, 32, 2046], [1, 1, 1, 1])
    run = ScaledRun(device, case, max_tokens=8)
    expected = run.run()
    assert_close(expected, *reference(case))
    elems = case.q_bits.size
    q_host, out_hosts = PinnedArray(elems, np.uint16), [PinnedArray(elems, np.uint16) for _ in range(2)]
    q_host.array[:] = case.q_bits.reshape(-1)
    q_dev, out_dev = run.q, run.out
    run.attention.attend_host(run.stream, q_host, out_hosts[0], q_dev, out_dev, run.pages, run.ids, case.slots, case.histories, case.cu)
    run.stream.synchronize()
    assert np.array_equal(bits_to_f32("bf16", out_hosts[0].array.copy()).reshape(expected.shape), expected)
    pipeline = HostPipeline(run.attention, run.stream)
    for step in range(5):
        out_hosts[step % 2].array[:] = 0
        ticket, *_ = pipeline.submit(q_host, out_hosts[step % 2], run.pages, run.ids, case.slots, case.histories, case.cu, case.layer)
        pipeline.wait(ticket)
        assert np.array_equal(bits_to_f32("bf16", out_hosts[step % 2].array.copy()).reshape(expected.shape), expected)
    pipeline.drain()
    assert device.check(run.stream) == 0


# ---- bidirectional block behind a scaled history ---------------------------------------------------------------------------
@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("windows", [[0] * 7, [4, 5, 6, 7, 8, 9, 10, 11]])
@pytest.mark.parametrize("hq,d,page", [(5, 128, 8), (5, 128, 16), (5, 256, 32), (8, 256, 16)])
def test_history_and_block_composite(device, code, windows, hq, d, page):
    """History partials of the sliced-Q map over scaled pages (per-token windows [begin, 12), two tasks), the block's partial
    in the range's last slot, one reduce: as over the other page types."""
    from khalamari_b200 import bidi_block_sdpa as bidi, sliced_q
    from khalamari_b200.device import Buffer, Dtype
    from khalamari_b200.sdpa import ExecutionVariant
    tokens, history = len(windows), 32
    case = make_scaled_case(91, code, "bf16", hq, 1, d, [history - tokens], [tokens], page=page)
    run = ScaledRun(device, case)
    rng = np.random.default_rng(92)
    (lk_bits, lk), (lv_bits, lv) = (round_to("bf16", rng.standard_normal((tokens, 1, d)).astype(np.float32)) for _ in range(2))
    config = sliced_q.Config(hq, 1, d, case.scale, page_bytes(1, page, d), run.io, run.layout, run.kv)
    execution = ExecutionVariant.sliced_q(config.sdpa_config(), 3, 8, 16, hq)
    shape = sliced_q.Shape(tokens, 1, 4)
    sizes = config.sizes(execution, shape)
    d_po, d_ps, d_pm = (Buffer.new_zeroed(device, n) for n in (
        sizes.partial_output_bytes, sizes.partial_output_stats_bytes, sizes.partial_output_stats_bytes))
    d_ranges, d_cu = (Buffer.from_slice(device, np.array(x, np.uint32)) for x in ([0, tokens], [0, 3]))
    visible = np.array([[w, 12] for w in windows], np.uint32).reshape(-1)
    templates = np.array([0, 0, 4, 0, 4, 12] + [0xFFFFFFFF] * 6, np.uint32)
    history_map = sliced_q.Compute(device, config, execution, shape)
    history_map.invoke_map(run.stream, sliced_q.MapBuffers(
        run.q, run.pages, Buffer.from_slice(device, np.full(tokens, case.slots[0], np.uint32)), run.ids,
        Buffer.from_slice(device, visible), d_ranges, Buffer.from_slice(device, templates), d_po, d_ps, d_pm), 0, tokens, 1, 3)
    bidi.Compute(device, bidi.Config(tokens, 8, hq, 1, d, case.scale, Dtype.Bfloat16)).invoke(
        run.stream, bidi.Shape(tokens, 1, 4), 1, bidi.Buffers(
            run.q, Buffer.from_slice(device, lk_bits), Buffer.from_slice(device, lv_bits), d_ranges, d_cu, d_ps, d_pm, d_po))
    history_map.invoke_reduce(run.stream, sliced_q.ReduceBuffers(d_po, d_ps, d_pm, d_ranges, d_cu, run.out), 1)
    out = run.read()
    # token t of the chunk sees its window's rows, then all of the block: as sequences of its own
    case.k = [np.concatenate([case.k[0][w:12], lk.astype(np.float64)]) for w in windows]
    case.v = [np.concatenate([case.v[0][w:12], lv.astype(np.float64)]) for w in windows]
    wide = 8 * hq > (32 if d == 128 else 24)
    expected, bound = reference(case, [(t, 0, len(k)) for t, k in enumerate(case.k)], wide=wide)
    assert_close(out, expected, bound)
