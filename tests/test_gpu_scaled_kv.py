"""Scaled 8-bit pages (``-m gpu``): quantising page write, page read-back and attention, against 64-bit restatements."""
import numpy as np
import pytest

from helpers import bits_to_f32, nan_bits, round_to
from scaled_helpers import CODES, ScaledRun, assert_close, make_scaled_case, page_bytes, planes, quantise, reference, values_of

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def device():
    from khalamari_b200.device import Device
    return Device(0)


def _dtype(name):
    from khalamari_b200.device import Dtype
    return {"bf16": Dtype.Bfloat16, "f16": Dtype.Float16, "int8": Dtype.Int8Scaled, "e4m3": Dtype.Fp8E4M3Scaled,
            "fp8": Dtype.Fp8E4M3FN}[name]


class Cache:
    """One pool and table with the write and read components over them."""

    def __init__(self, device, kind, io, hkv, d, page, table, pages, fill=0x55, ids_per_block=1, row_bytes=None):
        from khalamari_b200 import kv_page_read, kv_page_write
        from khalamari_b200.device import Buffer, Stream
        from khalamari_b200.request_page_table import GQAPageTableLayout

        self.device, self.hkv, self.d, self.page, self.io = device, hkv, d, page, io
        bytes_per_page = row_bytes or page_bytes(hkv, page, d)
        slots, layers, ids = table.shape
        self.layout = GQAPageTableLayout(slots, layers, ids // ids_per_block, ids_per_block)
        self.stream = Stream(device)
        self.pages = Buffer.from_slice(device, np.full(pages * bytes_per_page, fill, np.uint8))
        self.ids = Buffer.from_slice(device, table.astype(np.uint32).reshape(-1))
        config = kv_page_write.Config(hkv, d, bytes_per_page, _dtype(io), _dtype(kind))
        self.writer, self.reader = kv_page_write.Compute(device, config), kv_page_read.Compute(device, config)
        self.kvw, self.kvr, self.Buffer = kv_page_write, kv_page_read, Buffer

    def write(self, k_bits, v_bits, slots, tokens, active=None, layer=0, capacity=None):
        n = len(slots)
        self.held = [self.Buffer.from_slice(self.device, x) for x in
                     (k_bits, v_bits, np.asarray(slots, np.uint32), np.asarray(tokens, np.uint32))]
        self.writer.invoke(self.stream, self.kvw.Shape(n, self.layout), self.kvw.Buffers(self.pages, *self.held, self.ids),
                           n if active is None else active, layer)
        self.stream.synchronize()

    def read(self, slots, tokens, active=None, layer=0, canary=0x4228):
        n, row = len(slots), self.hkv * self.d
        outs = [self.Buffer.from_slice(self.device, np.full(n * row, canary, np.uint16)) for _ in range(2)]
        idx = [self.Buffer.from_slice(self.device, np.asarray(x, np.uint32)) for x in (slots, tokens)]
        self.reader.invoke(self.stream, self.kvr.Shape(n, self.layout),
                           self.kvr.Buffers(self.pages, *outs, *idx, self.ids), n if active is None else active, layer)
        self.stream.synchronize()
        return [o.read(0, n * row, np.uint16).reshape(n, self.hkv, self.d) for o in outs]

    def pool(self):
        return self.pages.read(0, self.pages.len_bytes(), np.uint8)


def _rows(rng, io, n, hkv, d, spread=8):
    x = rng.standard_normal((n, hkv, d)) * np.exp2(rng.integers(-spread, spread + 1, (n, hkv, 1)))
    return round_to(io, x.astype(np.float32))


@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("io", ["bf16", "f16"])
@pytest.mark.parametrize("hkv,d,page", [(1, 128, 8), (8, 128, 16), (3, 256, 8), (2, 256, 32), (5, 256, 16)])
def test_write_stores_the_restated_bytes_and_nothing_else(device, code, io, hkv, d, page):
    rng = np.random.default_rng(hkv * d + page)
    table = rng.permutation(40)[:2 * 3 * 5].reshape(2, 3, 5)  # two slots, three layers, five pages each
    cache = Cache(device, code, io, hkv, d, page, table, 41)
    tokens = np.concatenate([rng.permutation(5 * page)[:2 * page], np.arange(3, 3 + page + 2)])  # any order, odd starts
    slots = np.array([1] * (2 * page) + [0] * (page + 2))
    k_bits, k = _rows(rng, io, len(slots), hkv, d)
    v_bits, v = _rows(rng, io, len(slots), hkv, d)
    k_bits[3], k[3] = 0, 0  # a row of zeros
    expected = cache.pool().copy()
    codes, scales = planes(expected, hkv, page, d)
    active = len(slots) - 2  # the last rows stay unwritten
    for plane, x in enumerate((k, v)):
        c, b = quantise(x, code)
        at = table[slots[:active], 2, tokens[:active] // page]
        codes[at, plane, :, tokens[:active] % page] = c[:active]
        scales[at, :, plane, tokens[:active] % page] = b[:active]
    cache.write(k_bits, v_bits, slots, tokens, active, layer=2)
    assert device.check(cache.stream) == 0
    got = cache.pool()
    assert np.array_equal(got, expected)


@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("io", ["bf16", "f16"])
def test_rows_at_the_edges_of_the_range(device, code, io):
    """Every exponent of the source type, values that round up to the next power of two, ties, subnormals."""
    d, page = 128, 16
    specials = []
    low, high = (-133, 127) if io == "bf16" else (-24, 15)
    for k in range(low, high + 1):
        # (the largest values: a row whose codes round up may stand for 2^(k + 1), beyond the type's range)
        for m in (1.0, 1.75, 1.7578125, 1.984375, 1.9921875, 1.5):
            row = np.zeros(d, np.float64)
            row[0] = m * 2.0 ** k
            row[1:8] = [-row[0], row[0] / 2, row[0] / 254, row[0] * 3 / 254, row[0] / 896, row[0] * 2.0 ** -9, row[0] * 2.0 ** -17]
            specials.append(row)
    x = np.array(specials)
    most = float(np.float32(3.3895313892515355e38)) if io == "bf16" else 65504.0
    x = np.clip(x, -most, most).astype(np.float32)
    bits, x = round_to(io, x)
    n = len(x)
    bits, x = bits.reshape(n, 1, d), x.reshape(n, 1, d)
    cache = Cache(device, code, io, 1, d, page, np.arange(-(-n // page)).reshape(1, 1, -1), -(-n // page))
    cache.write(bits, bits[::-1].copy(), np.zeros(n), np.arange(n))
    codes, scales = planes(cache.pool(), 1, page, d)
    at = np.arange(n)
    c, b = quantise(x, code)
    got = codes[at // page, 0, 0, at % page]
    assert np.array_equal(scales[at // page, 0, 0, at % page], b[:, 0])
    # (a zero may carry either sign)
    assert np.array_equal(values_of(got, b[:, 0], code), values_of(c[:, 0], b[:, 0], code))
    k_out, _ = cache.read(np.zeros(n), at)
    expected = np.clip(values_of(c, b, code), -most, most)
    assert np.array_equal(bits_to_f32(io, k_out), round_to(io, expected.astype(np.float32))[1])
    assert device.check(cache.stream) == 0


@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("io", ["bf16", "f16"])
@pytest.mark.parametrize("d", [128, 256])
@pytest.mark.parametrize("value", [np.nan, np.inf, -np.inf])
def test_rows_that_are_not_finite_read_back_as_nan(device, code, io, d, value):
    rng = np.random.default_rng(2)
    hkv, page, n = 2, 16, 5
    k_bits, k = _rows(rng, io, n, hkv, d)
    v_bits, v = _rows(rng, io, n, hkv, d)
    bad, _ = round_to(io, np.array([value], np.float32))
    k_bits[1, 0, d - 1] = bad[0]
    v_bits[3, 1, 7] = bad[0]
    cache = Cache(device, code, io, hkv, d, page, np.zeros((1, 1, 1)), 1)
    cache.write(k_bits, v_bits, np.zeros(n), np.arange(n))
    codes, scales = planes(cache.pool(), hkv, page, d)
    for token, head in ((1, 0), (3, 1)):
        assert np.all(scales[0, head, :, token] == 255) and not codes[0, :, head, token].any()
    assert np.count_nonzero(scales[0, :, :, :n] == 255) == 4
    for out, x in zip(cache.read(np.zeros(n), np.arange(n)), (k, v)):
        got = bits_to_f32(io, out)
        assert np.isnan(got[1, 0]).all() and np.isnan(got[3, 1]).all()
        good = np.ones((n, hkv), bool)
        good[1, 0] = good[3, 1] = False
        assert np.array_equal(got[good], values_of(*quantise(x[good], code), code).astype(np.float32))


@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("hkv,d,page", [(1, 128, 8), (8, 128, 16), (2, 256, 32), (5, 256, 16)])
def test_read_gathers_any_order_and_leaves_the_rest(device, code, hkv, d, page):
    rng = np.random.default_rng(3)
    table = rng.permutation(12).reshape(2, 2, 3)
    cache = Cache(device, code, "bf16", hkv, d, page, table, 12, ids_per_block=3)
    n = 3 * page
    bits = [_rows(rng, "bf16", 2 * n, hkv, d) for _ in range(2)]
    slots, tokens = np.repeat([0, 1], n), np.tile(np.arange(n), 2)
    cache.write(bits[0][0], bits[1][0], slots, tokens, layer=1)
    pick = rng.integers(0, 2 * n, 2 * page + 3)  # repeats among them
    outs = cache.read(slots[pick], tokens[pick], active=len(pick) - 3, layer=1)
    for out, (_, x) in zip(outs, bits):
        expected = values_of(*quantise(x, code), code)[pick].astype(np.float32)  # exact in bf16
        assert np.array_equal(bits_to_f32("bf16", out[:-3]), expected[:-3])
        assert np.all(out[-3:] == 0x4228)
    assert device.check(cache.stream) == 0


@pytest.mark.parametrize("kind,d,elem", [("bf16", 128, 2), ("bf16", 9, 2), ("fp8", 256, 1), ("fp8", 9, 1)])
def test_read_inverts_the_write_of_the_other_page_types(device, kind, d, elem):
    rng = np.random.default_rng(4)
    hkv, page, n = 2, 4, 11
    cache = Cache(device, kind, "bf16", hkv, d, page, np.array([[[2, 0, 1]]]), 3, row_bytes=2 * hkv * page * d * elem)
    bits, x = _rows(rng, "bf16", n, hkv, d, spread=3)
    bits[2, 1, 3] = nan_bits("bf16")
    cache.write(bits, bits[::-1].copy(), np.zeros(n), np.arange(n))
    k_out, v_out = cache.read(np.zeros(n), np.arange(n))
    if kind == "bf16":
        assert np.array_equal(k_out, bits) and np.array_equal(v_out, bits[::-1])
    else:
        import oracle
        back = oracle.fp8_to_bf16_bits(oracle.fp8_from_bf16_bits(bits.reshape(-1))).reshape(bits.shape)
        a, b = bits_to_f32("bf16", k_out), oracle.bf16_bits_to_f32(back)
        assert np.array_equal(a, b, equal_nan=True) and np.isnan(a[2, 1, 3])


@pytest.mark.parametrize("code", CODES)
def test_metadata_beyond_the_tables_is_reported_and_skipped(device, code):
    from khalamari_b200 import abi
    rng = np.random.default_rng(6)
    hkv, d, page = 2, 128, 8
    table = np.array([[[0, 9]]])  # page 9 is beyond a pool of two pages
    bits, x = _rows(rng, "bf16", 3, hkv, d)
    for slots, tokens, word in (([0, 7, 0], [0, 0, 1], 4), ([0, 0, 0], [0, 16, 1], 4), ([0, 0, 0], [0, 8, 1], 2)):
        cache = Cache(device, code, "bf16", hkv, d, page, table, 2)
        before = cache.pool()
        cache.write(bits, bits, slots, tokens)
        with pytest.raises(abi.KhError, match=f"0x{word:x}"):
            device.check(cache.stream)
        codes, scales = planes(cache.pool(), hkv, page, d)
        assert np.array_equal(codes[0, 0, :, :2], quantise(x[[0, 2]], code)[0].transpose(1, 0, 2))
        assert np.array_equal(cache.pool()[before.size // 2:], before[before.size // 2:])
        k_out, _ = cache.read(slots, tokens)
        with pytest.raises(abi.KhError, match=f"0x{word:x}"):
            device.check(cache.stream)
        assert np.all(k_out[1] == 0x4228)
        assert np.array_equal(bits_to_f32("bf16", k_out[[0, 2]]), values_of(*quantise(x[[0, 2]], code), code).astype(np.float32))


def test_write_and_read_refuse_what_they_cannot_do(device):
    from khalamari_b200 import abi, kv_page_read, kv_page_write
    from khalamari_b200.device import Buffer
    cache = Cache(device, "int8", "bf16", 2, 128, 16, np.zeros((1, 1, 1)), 1)
    good = [Buffer.new_zeroed(device, 4 * 2 * 128 * 2) for _ in range(2)] + [Buffer.new_zeroed(device, 16) for _ in range(2)]
    shape = kv_page_read.Shape(4, cache.layout)
    odd = Buffer.wrap(device, good[0].ref.ptr + 8, good[0].len_bytes() - 8)

    def call(buffers, active=4, layer=0, shape=shape):
        cache.reader.invoke(cache.stream, shape, kv_page_read.Buffers(*buffers), active, layer)

    buffers = [cache.pages, *good, cache.ids]
    for at, name in enumerate(("pages", "flat_k", "flat_v", "req_slots", "flat_token_indices", "page_ids")):
        replaced = list(buffers)
        replaced[at] = Buffer.wrap(device, buffers[at].ref.ptr, 2)
        with pytest.raises(abi.InvalidArgument, match=name):
            call(replaced)
    for active in (0, 5):
        with pytest.raises(abi.InvalidArgument, match="num_active_token_reads"):
            call(buffers, active)
    with pytest.raises(abi.InvalidArgument, match="page_table_index"):
        call(buffers, layer=1)
    tight = kv_page_read.Shape(3, cache.layout)
    with pytest.raises(abi.InvalidArgument, match="16-byte aligned"):
        call([cache.pages, odd, *buffers[2:]], 3, shape=tight)
    with pytest.raises(abi.InvalidArgument, match="16-byte aligned"):
        cache.writer.invoke(cache.stream, kv_page_write.Shape(3, cache.layout),
                            kv_page_write.Buffers(cache.pages, odd, *buffers[2:]), 3)


# ---- attention ------------------------------------------------------------------------------------------------------
DECODE = [
    # hq, hkv, d, page, contexts
    (8, 8, 128, 16, [1, 2, 15, 16, 17, 31, 33]),
    (64, 8, 128, 16, [700, 33, 1500, 1]),
    (8, 1, 128, 8, [9, 64, 127, 300]),
    (5, 1, 128, 16, [129, 257]),
    (28, 4, 128, 8, [100, 47]),
    (16, 2, 256, 16, [128, 517, 1024, 2048]),
    (6, 1, 256, 32, [31, 32, 33, 500]),
    (12, 4, 256, 8, [7, 90]),
    (16, 1, 128, 16, [300, 40]),     # a group of 16 heads: two rows of n-tiles
    (24, 1, 256, 16, [200, 21]),
]


@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("io", ["bf16", "f16"])
@pytest.mark.parametrize("hq,hkv,d,page,contexts", DECODE)
def test_decode_matches_the_64_bit_restatement(device, code, io, hq, hkv, d, page, contexts):
    case = make_scaled_case(hq + d, code, io, hq, hkv, d, [c - 1 for c in contexts], [1] * len(contexts), page=page,
                            layers=2, layer=1)
    assert_close(ScaledRun(device, case).run(), *reference(case))


@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("io", ["bf16", "f16"])
@pytest.mark.parametrize("hq,hkv,d,page,histories,q_lens", [
    (24, 4, 256, 16, [300, 61], [4, 4]),
    (64, 8, 128, 16, [200, 17, 0], [2, 3, 4]),
    (16, 2, 128, 8, [90, 0], [24, 19]),
    (16, 2, 256, 32, [0], [45]),
    (4, 4, 128, 16, [33, 5], [70, 1]),
    (7, 1, 256, 8, [12], [37]),
    (8, 1, 128, 16, [500], [150]),
])
def test_several_tokens_match_the_64_bit_restatement(device, code, io, hq, hkv, d, page, histories, q_lens):
    case = make_scaled_case(hq * d, code, io, hq, hkv, d, histories, q_lens, page=page)
    run = ScaledRun(device, case, max_tokens=256)
    assert_close(run.run(), *reference(case, wide=run.wide()))


def _wild(low, high):
    return lambda rng, tokens, heads: np.exp2(rng.uniform(low, high, (tokens, heads)))


@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("d", [128, 256])
def test_rows_of_very_different_sizes(device, code, d):
    """V rows whose scales differ by 2^24 and K rows by 2^8, some of them zero: a weight is rounded relative to the
    largest weight of its Q row, whatever single rows are scaled by."""
    def some_zero(rng, tokens, heads):
        return _wild(-12, 12)(rng, tokens, heads) * (rng.random((tokens, heads)) > 0.2)
    case = make_scaled_case(3, code, "bf16", 8, 2, d, [399, 40, 0], [1, 2, 1], k_scale=_wild(-6, 2), v_scale=some_zero)
    assert_close(ScaledRun(device, case).run(), *reference(case))


@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("slice_tokens", [16, 40, 64, 333, 512])
def test_forced_slices_of_one_chain(device, code, slice_tokens):
    """Slices of any length, aligned to tiles or not: neighbours of one CTA are merged before they are published."""
    case = make_scaled_case(8, code, "bf16", 16, 2, 128, [1999, 700, 64], [1, 1, 1])
    run = ScaledRun(device, case, max_tokens=512)
    variant = next(v for v in run.attention.selector.variants() if v.kind == 0 and v.thread_block.max_q_tokens == 1)
    selection = run.attention.select_partitioned(variant, slice_tokens, False, case.histories, case.cu)
    assert_close(run.run(selection), *reference(case), f"slices of {slice_tokens}")


def test_many_short_sequences(device):
    rng = np.random.default_rng(12)
    contexts = rng.integers(1, 60, 400).tolist()
    case = make_scaled_case(13, "int8", "bf16", 8, 2, 128, [c - 1 for c in contexts], [1] * len(contexts))
    assert_close(ScaledRun(device, case).run(), *reference(case))


@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("d,page", [(128, 16), (128, 8), (256, 32)])
def test_windows_and_rows_that_see_nothing(device, code, d, page):
    """Per-token visible ranges of the sliced-Q map: sliding windows, empty ones, tiles of which only some rows see a
    token. Pages below a window are unallocated (garbage ids): only what is visible is fetched."""
    from khalamari_b200 import sliced_q
    from khalamari_b200.device import Buffer
    from khalamari_b200.sdpa import ExecutionVariant
    hq, hkv, tokens, context = 4, 2, 6, 200
    case = make_scaled_case(21, code, "bf16", hq, hkv, d, [context - tokens], [tokens], page=page)
    first = 72
    case.table[case.slots[0], 0, :first // page] = 0xFFFFFF00
    run = ScaledRun(device, case)
    config = sliced_q.Config(hq, hkv, d, case.scale, page_bytes(hkv, page, d), run.io, run.layout, run.kv)
    windows = [(72, 75), (100, 100), (80, 161), (199, 200), (73, 200), (150, 90)]
    visible = np.array(windows, np.uint32)
    execution = ExecutionVariant.sliced_q(config.sdpa_config(), 3, 8, 16, 2)
    for splits in ([(0, 200)], [(0, 100), (100, 200)], [(0, 40), (40, 77), (77, 200)]):
        shape = sliced_q.Shape(tokens, 1, 4)
        sizes = config.sizes(execution, shape)
        compute = sliced_q.Compute(device, config, execution, shape)
        templates = np.full((4, 3), 0xFFFFFFFF, np.uint32)
        templates[:len(splits)] = [(0, b, e) for b, e in splits]
        d_slots = Buffer.from_slice(device, np.full(tokens, case.slots[0], np.uint32))
        d_visible, d_ranges = Buffer.from_slice(device, visible), Buffer.from_slice(device, np.array([0, tokens], np.uint32))
        d_templates = Buffer.from_slice(device, templates)
        d_cu = Buffer.from_slice(device, np.array([0, len(splits)], np.uint32))
        d_po, d_ps, d_pm = (Buffer.new_zeroed(device, n) for n in (
            sizes.partial_output_bytes, sizes.partial_output_stats_bytes, sizes.partial_output_stats_bytes))
        compute.invoke_map(run.stream, sliced_q.MapBuffers(run.q, run.pages, d_slots, run.ids, d_visible, d_ranges,
                                                           d_templates, d_po, d_ps, d_pm), 0, tokens, 1, len(splits))
        compute.invoke_reduce(run.stream, sliced_q.ReduceBuffers(d_po, d_ps, d_pm, d_ranges, d_cu, run.out), 1)
        out = run.read()
        expected, bound = reference(case, [(0, b, e) for b, e in windows])
        assert_close(out, expected, bound, f"splits {splits}")
        assert not out[1].any() and not out[5].any()


@pytest.mark.parametrize("code", CODES)
def test_rows_that_are_not_finite_reach_only_the_queries_that_see_them(device, code):
    case = make_scaled_case(30, code, "bf16", 8, 2, 128, [60, 60], [8, 8])
    codes, scales = planes(case.pool, 2, 16, 128)
    page = case.table[case.slots[0], 0, 64 // 16]
    scales[page, 1, :, 64 % 16] = 255  # token 64 of request 0, KV head 1: seen by its queries 4..7 only
    codes[page, :, 1, 64 % 16] = 0
    run = ScaledRun(device, case, max_tokens=32)
    run.plan()
    run.record()
    out = run.read()
    expected, bound = reference(case)
    hidden = np.zeros(out.shape[:2], bool)
    hidden[4:8, 4:] = True
    assert np.isnan(out[hidden]).all()
    assert_close(out[~hidden], expected[~hidden], bound[~hidden])


def test_large_offsets_in_a_pool_beyond_4_gib(device):
    """A pool of more than 2^32 bytes whose used pages lie at its end."""
    import torch
    case = make_scaled_case(40, "int8", "bf16", 16, 2, 256, [77, 300], [1, 1])
    per_page = page_bytes(2, 16, 256)
    used = len(case.pool) // per_page
    pages = (5 << 30) // per_page
    big = torch.zeros(pages * per_page, dtype=torch.uint8, device="cuda")
    big[-len(case.pool):] = torch.from_numpy(case.pool).cuda()
    case.table[case.table != 0xFFFFFFFF] += pages - used
    run = ScaledRun(device, case)
    run.pages = type(run.pages).wrap(device, big.data_ptr(), big.numel())
    torch.cuda.synchronize()
    assert_close(run.run(), *reference(case))


def test_a_page_id_beyond_the_pool_is_reported(device):
    from khalamari_b200 import abi
    case = make_scaled_case(41, "e4m3", "bf16", 8, 2, 128, [40], [1])
    case.table[case.slots[0], 0, 1] = 10 ** 6
    run = ScaledRun(device, case)
    run.plan()
    run.record()
    with pytest.raises(abi.KhError, match="page id"):
        run.stream.synchronize()
        device.check(run.stream)


def test_unaligned_buffers_and_the_one_launch_form_are_refused(device):
    from khalamari_b200 import abi
    from khalamari_b200.device import Buffer
    case = make_scaled_case(42, "int8", "bf16", 8, 2, 128, [40], [1])
    run = ScaledRun(device, case)
    run.plan()
    run.attention.fused = True
    with pytest.raises(abi.InvalidArgument, match="one-launch"):
        run.record()
    run.attention.fused = False
    pages = run.pages
    run.pages = Buffer.wrap(device, pages.ref.ptr + 8, pages.len_bytes() - 8)
    with pytest.raises(abi.InvalidArgument, match="kv_pages must be 16-byte aligned"):
        run.record()
    run.pages = pages
    run.q = Buffer.wrap(device, run.q.ref.ptr + 2, run.q.len_bytes())
    with pytest.raises(abi.InvalidArgument, match="q must be 16-byte aligned"):
        run.record()


def test_unaligned_direct_output_is_refused(device):
    from khalamari_b200 import abi
    from khalamari_b200.device import Buffer
    case = make_scaled_case(43, "int8", "bf16", 16, 2, 128, [0], [40])
    run = ScaledRun(device, case, max_tokens=512)
    run.plan()
    if not run.attention.metadata.direct_output():
        pytest.skip("this batch is not written directly")
    run.out = Buffer.wrap(device, run.out.ref.ptr + 2, run.out.len_bytes() - 2)
    with pytest.raises(abi.InvalidArgument, match="output must be 16-byte aligned"):
        run.record()


@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("d", [128, 256])
@pytest.mark.parametrize("hq,q_len", [(16, 1), (32, 1), (16, 2), (32, 3), (64, 1), (32, 40)])
def test_groups_of_many_heads(device, code, d, hq, q_len):
    """One KV head for 16 to 64 Q heads: tasks of 16 rows and more, and groups cut into ranges of heads."""
    case = make_scaled_case(hq + q_len, code, "bf16", hq, 1, d, [700 - q_len, 33], [q_len, q_len])
    run = ScaledRun(device, case, max_tokens=512)
    out = run.run()
    assert_close(out, *reference(case, wide=run.wide()))


@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("hq,hkv,d,contexts", [(64, 8, 128, [3000, 17, 1024, 640]), (16, 2, 256, [900, 4100, 33])])
def test_the_shared_array_form_gives_the_same_bits(device, code, hq, hkv, d, contexts):
    from khalamari_b200 import sliced_kv
    case = make_scaled_case(91, code, "bf16", hq, hkv, d, [c - 1 for c in contexts], [1] * len(contexts))
    run = ScaledRun(device, case)
    expected = run.run()
    meta = run.attention.metadata
    shape = meta.replay_shape()
    compute = run.attention._sliced_kv(shape, meta.variant())
    run.out.write(0, np.full(run.out_rows * run.row, run.canary, np.uint16))
    compute.invoke_attend_static(
        run.stream, sliced_kv.StaticBuffers(run.q, run.pages, meta.req_slots(), run.ids, meta.sdpa_map_task_templates(),
                                            meta.cu_sdpa_partial_outputs(), run.out),
        case.layer, shape.num_tokens, shape.num_sdpa_map_task_templates)
    assert np.array_equal(expected, run.read())


@pytest.mark.parametrize("code", CODES)
def test_append_then_attend_over_several_steps(device, code):
    """The operators together, as a serving loop has them: each step writes the new token's rows and attends; at the
    end the whole cache is read back. An append changes no byte of earlier tokens."""
    from khalamari_b200 import kv_page_write
    from khalamari_b200.device import Buffer
    rng = np.random.default_rng(50)
    hq, hkv, d, page, steps = 8, 2, 128, 16, 20
    case = make_scaled_case(51, code, "bf16", hq, hkv, d, [28 + steps, 3 + steps], [1, 1], page=page)
    start = [29, 4]
    case.k, case.v = [k[:n] for k, n in zip(case.k, start)], [v[:n] for v, n in zip(case.v, start)]
    run = ScaledRun(device, case, max_tokens=8)
    config = kv_page_write.Config(hkv, d, page_bytes(hkv, page, d), run.io, run.kv)
    writer = kv_page_write.Compute(device, config)
    d_k, d_v = (Buffer.new_zeroed(device, 2 * hkv * d * 2) for _ in range(2))
    d_slots, d_tokens = Buffer.from_slice(device, np.array(case.slots, np.uint32)), Buffer.new_zeroed(device, 8)
    for step in range(steps):
        before = run.pages.read(0, run.pages.len_bytes(), np.uint8)
        (k_bits, k), (v_bits, v) = (_rows(rng, "bf16", 2, hkv, d, spread=2) for _ in range(2))
        at = [n + step for n in start]
        d_k.write(0, k_bits)
        d_v.write(0, v_bits)
        d_tokens.write(0, np.array(at, np.uint32))
        q_bits, _ = round_to("bf16", rng.standard_normal((2, hq, d)).astype(np.float32))
        case.q_bits, case.histories = q_bits, at
        run.q.write(0, q_bits)
        for r in range(2):
            case.k[r] = np.concatenate([case.k[r], values_of(*quantise(k[r:r + 1], code), code)])
            case.v[r] = np.concatenate([case.v[r], values_of(*quantise(v[r:r + 1], code), code)])
        writer.invoke(run.stream, kv_page_write.Shape(2, run.layout),
                      kv_page_write.Buffers(run.pages, d_k, d_v, d_slots, d_tokens, run.ids), 2)
        assert_close(run.run(), *reference(case), f"step {step}")
        after = run.pages.read(0, run.pages.len_bytes(), np.uint8)
        assert np.count_nonzero(before != after) <= 2 * hkv * 2 * (d + 1)
    from khalamari_b200 import kv_page_read
    n = [len(k) for k in case.k]
    outs = [Buffer.new_zeroed(device, sum(n) * hkv * d * 2) for _ in range(2)]
    kv_page_read.Compute(device, config).invoke(
        run.stream, kv_page_read.Shape(sum(n), run.layout),
        kv_page_read.Buffers(run.pages, *outs, Buffer.from_slice(device, np.repeat(case.slots, n).astype(np.uint32)),
                             Buffer.from_slice(device, np.concatenate([np.arange(x) for x in n]).astype(np.uint32)), run.ids),
        sum(n))
    run.stream.synchronize()
    for out, x in zip(outs, (case.k, case.v)):
        got = bits_to_f32("bf16", out.read(0, sum(n) * hkv * d, np.uint16)).reshape(-1, hkv, d)
        assert np.array_equal(got, np.concatenate(x).astype(np.float32))


@pytest.mark.parametrize("code", CODES)
def test_captured_step_replays_for_other_batches(device, code):
    """Write and attention captured into one CUDA graph, replayed with other batches and new rows."""
    import torch

    from khalamari_b200 import kv_page_write
    from khalamari_b200.device import Buffer, Stream
    rng = np.random.default_rng(60)
    hq, hkv, d = 16, 2, 128
    case = make_scaled_case(61, code, "bf16", hq, hkv, d, [299, 610, 59, 1000], [1] * 4)
    run = ScaledRun(device, case, max_tokens=8)
    torch_stream = torch.cuda.Stream()
    run.stream = Stream(device, torch_stream.cuda_stream)
    variant = next(v for v in run.attention.selector.variants() if v.kind == 0 and v.thread_block.max_q_tokens == 1)
    writer = kv_page_write.Compute(device, kv_page_write.Config(hkv, d, page_bytes(hkv, 16, d), run.io, run.kv))
    d_k, d_v = (Buffer.new_zeroed(device, 4 * hkv * d * 2) for _ in range(2))
    d_slots, d_tokens = Buffer.new_zeroed(device, 16), Buffer.new_zeroed(device, 16)
    q = Buffer.new_zeroed(device, 4 * run.row * 2)

    def plan(order):
        histories = [case.histories[r] for r in order]
        selection = run.attention.select_partitioned(variant, 256, False, histories, [0, 1, 2, 3, 4], 4)
        run.attention.prepare([case.slots[r] for r in order], histories, [0, 1, 2, 3, 4], 4, run.stream, selection)

    def step():
        writer.invoke(run.stream, kv_page_write.Shape(4, run.layout),
                      kv_page_write.Buffers(run.pages, d_k, d_v, d_slots, d_tokens, run.ids), 4)
        run.attention.record_replay(run.stream, q, run.pages, run.ids, run.out, 0)

    plan([0, 1, 2, 3])
    d_slots.write(0, np.array(case.slots, np.uint32))
    d_tokens.write(0, np.array(case.histories, np.uint32))
    graph = torch.cuda.CUDAGraph()
    step()
    torch_stream.synchronize()
    with torch.cuda.graph(graph, stream=torch_stream):
        step()
    for order in ([2, 0, 3, 1], [1, 3, 2, 0]):
        plan(order)
        (k_bits, k), (v_bits, v) = (_rows(rng, "bf16", 4, hkv, d, spread=2) for _ in range(2))
        torch_stream.synchronize()
        d_k.write(0, k_bits)
        d_v.write(0, v_bits)
        d_slots.write(0, np.array([case.slots[r] for r in order], np.uint32))
        d_tokens.write(0, np.array([case.histories[r] for r in order], np.uint32))
        q.write(0, case.q_bits[order])
        for i, r in enumerate(order):
            case.k[r][-1:] = values_of(*quantise(k[i:i + 1], code), code)
            case.v[r][-1:] = values_of(*quantise(v[i:i + 1], code), code)
        with torch.cuda.stream(torch_stream):
            graph.replay()
        out = run.read()
        expected, bound = reference(case)
        assert_close(out, expected[order], bound[order], f"order {order}")


def test_prefill_and_decode_in_one_call(device):
    from khalamari_b200.device import Buffer
    from khalamari_b200.gqa import GQACore, MixedBatchAttention
    case = make_scaled_case(70, "int8", "bf16", 16, 2, 128, [40, 0, 333, 12], [30, 17, 1, 1])
    run = ScaledRun(device, case, max_tokens=64)
    mixed = MixedBatchAttention(device, GQACore(128, 16, 2, case.scale), run.io, page_bytes(2, 16, 128), run.layout, 64,
                                kv_dtype=run.kv)
    mixed.prepare(case.slots, case.histories, case.cu, run.stream)
    assert len(mixed.plan) == 2
    tokens = len(case.q_bits)
    q = Buffer.from_slice(device, case.q_bits)
    mixed.record_sdpa(run.stream, q, run.pages, run.ids, Buffer.wrap(device, run.out.ref.ptr, tokens * run.row * 2))
    assert_close(run.read(), *reference(case, wide=True))


# ---- wide Q tiles -----------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("io", ["bf16", "f16"])
@pytest.mark.parametrize("d,hq,hkv,page,histories,q_lens", [
    (128, 16, 2, 16, [700, 0, 133], [200, 129, 49]),   # odd numbers of tiles: pairs that straddle two requests
    (128, 32, 8, 8, [300], [333]),                     # a group of four heads, 32-token tiles
    (128, 12, 2, 16, [61, 5], [97, 64]),               # a group of six: 96 of 128 rows
    (128, 8, 1, 16, [2000], [40]),                     # few tiles: the KV range is cut
    (128, 5, 1, 8, [0], [300]),
    (256, 16, 2, 16, [300, 0], [100, 33]),
    (256, 12, 2, 8, [61, 5], [97, 64]),
    (256, 4, 4, 32, [200], [170]),
    (256, 8, 1, 32, [1500], [24]),
])
def test_wide_tiles_match_the_64_bit_restatement(device, code, io, d, hq, hkv, page, histories, q_lens):
    case = make_scaled_case(hq + page, code, io, hq, hkv, d, histories, q_lens, page=page)
    run = ScaledRun(device, case, max_tokens=512)
    out = run.run()
    assert run.wide()
    assert_close(out, *reference(case, wide=True))


@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("d,hq,hkv,page", [(128, 32, 8, 16), (128, 32, 8, 8), (256, 16, 4, 16), (256, 16, 4, 32)])
def test_many_ragged_wide_tiles_follow_one_another(device, code, d, hq, hkv, page):
    """Several tasks a CTA, most of them ending inside a step, some within its first 16 tokens: rings run on from task to task."""
    rng = np.random.default_rng(84)
    q_lens = rng.integers(9, 48, 120).tolist()
    histories = [0 if i % 4 == 0 else int(rng.integers(1, 200)) for i in range(120)]
    case = make_scaled_case(85, code, "bf16", hq, hkv, d, histories, q_lens, page=page)
    run = ScaledRun(device, case)
    out = run.run()
    assert run.wide()
    assert_close(out, *reference(case, wide=True))
    for _ in range(4):
        run.record()
        assert np.array_equal(out, run.read())


@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("d", [128, 256])
@pytest.mark.parametrize("io,low,high", [("bf16", -40, 40), ("f16", -14, 11)])
def test_wide_tiles_over_rows_of_very_different_sizes(device, code, d, io, low, high):
    """V rows whose scales differ by up to 2^80 (f16: up to its whole range), some of them zero."""
    def some_zero(rng, tokens, heads):
        return _wild(low, high)(rng, tokens, heads) * (rng.random((tokens, heads)) > 0.2)
    case = make_scaled_case(80, code, io, 16, 2, d, [200, 0], [64, 80], k_scale=_wild(-6, 1), v_scale=some_zero)
    assert_close(ScaledRun(device, case, max_tokens=256).run(), *reference(case, wide=True))


@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("io", ["bf16", "f16"])
@pytest.mark.parametrize("d", [128, 256])
def test_wide_tiles_and_rows_that_are_not_finite(device, code, io, d):
    case = make_scaled_case(81, code, io, 16, 2, d, [300, 150], [64, 40])
    codes, scales = planes(case.pool, 2, 16, d)
    at = 330  # a token of request 0's own chunk, KV head 1: seen by its queries from number 30 on
    page = case.table[case.slots[0], 0, at // 16]
    scales[page, 1, :, at % 16] = 255
    codes[page, :, 1, at % 16] = 0
    run = ScaledRun(device, case, max_tokens=256)
    run.plan()
    run.record()
    out = run.read()
    expected, bound = reference(case, wide=True)
    hidden = np.zeros(out.shape[:2], bool)
    hidden[30:64, 8:] = True
    assert np.isnan(out[hidden]).all()
    assert_close(out[~hidden], expected[~hidden], bound[~hidden])


@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("d,page", [(128, 8), (128, 16), (256, 8), (256, 32)])
def test_wide_tiles_with_windows(device, code, d, page):
    """Direct output with per-token visible ranges: windows of different lengths, empty ones, unallocated pages below."""
    from khalamari_b200 import sliced_q
    from khalamari_b200.device import Buffer
    from khalamari_b200.sdpa import ExecutionVariant
    hq, hkv, tokens, context = 16, 2, 32, 500
    case = make_scaled_case(82, code, "bf16", hq, hkv, d, [context - tokens], [tokens], page=page)
    case.table[case.slots[0], 0, :200 // page] = 0xFFFFFF00
    run = ScaledRun(device, case)
    config = sliced_q.Config(hq, hkv, d, case.scale, page_bytes(hkv, page, d), run.io, run.layout, run.kv)
    windows = [(200 + 7 * i, 200 + 7 * i + (0 if i % 5 == 3 else 40 + 3 * i)) for i in range(tokens)]
    execution = ExecutionVariant.sliced_q(config.sdpa_config(), 3, 16, 16, 8)
    shape = sliced_q.Shape(tokens, 2, 2)
    compute = sliced_q.Compute.new_direct(device, config, execution, shape)
    buffers = [Buffer.from_slice(device, np.array(x, np.uint32)) for x in (
        [case.slots[0]] * tokens, windows, [(0, 16), (16, 32)], [(0, 0, context), (1, 0, context)])]
    compute.invoke_direct(run.stream, sliced_q.DirectBuffers(run.q, run.pages, buffers[0], run.ids, *buffers[1:], run.out), 0, tokens, 2)
    out = run.read()
    expected, bound = reference(case, [(0, b, e) for b, e in windows], wide=True)
    assert_close(out, expected, bound)
    assert not out[3].any()
