"""One sequence over scaled 8-bit pages split in token order over several ranks (``-m gpu``), emulated on one GPU: the
ranks run one after another, each over a pool of its own pages, and their records are merged as an exchange leaves them
(kernels that wait for one another must not share a GPU, so other ranks' rows are delivered by the host)."""
import numpy as np
import pytest

from helpers import bits_to_f32
from scaled_helpers import CODES, ScaledRun, assert_close, make_scaled_case, planes, quantise, reference

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def device():
    from khalamari_b200.device import Device
    return Device(0)


def _local(full, begin, end, seed, broken=None):
    """The tokens [begin, end) of ``full``'s one sequence as a rank holds them. ``broken``: (token, KV head) whose scale
    bytes mark a row that is not finite."""
    n = max(end - begin, 1)
    case = make_scaled_case(seed, full.code, full.dtype_name, full.hq, full.hkv, full.d, [n - 1], [1], page=full.page, scale=full.scale)
    case.q_bits = full.q_bits
    codes, scales = planes(case.pool, full.hkv, full.page, full.d)
    tokens = np.arange(end - begin)
    at, row = case.table[case.slots[0], 0, tokens // full.page], tokens % full.page
    for plane, values in enumerate((full.k[0], full.v[0])):
        c, b = quantise(values[begin:end], full.code)  # (values that codes stand for: they come back exactly)
        codes[at, plane, :, row] = c
        scales[at, :, plane, row] = b
    if broken is not None and begin <= broken[0] < end:
        token, head = broken[0] - begin, broken[1]
        page = case.table[case.slots[0], 0, token // full.page]
        scales[page, head, :, token % full.page] = 255
        codes[page, :, head, token % full.page] = 0
    return case


def _full(code, hq, hkv, d, context):
    return make_scaled_case(7, code, "bf16", hq, hkv, d, [context - 1], [1])


def _check(out, full, broken):
    expected, bound = reference(full)
    hidden = np.zeros(out.shape[:2], bool)
    if broken is not None:
        group = full.hq // full.hkv
        hidden[:, broken[1] * group:(broken[1] + 1) * group] = True
    assert np.isnan(out[hidden]).all()
    # (the bound counts one rounding to bf16; the merges add f32 roundings only, far below its hundredth of slack)
    assert_close(out[~hidden], expected[~hidden], bound[~hidden])


@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("hq,hkv,d", [(16, 2, 128), (16, 2, 256), (12, 1, 256)])
@pytest.mark.parametrize("world,context,partition,broken", [
    (2, 3000, 256, None), (4, 3000, 64, None), (3, 40, 64, None),
    (1, 3000, 256, (1700, 0)), (2, 3000, 256, (2990, 0)), (4, 3000, 64, (5, 0)),
])
def test_ranks_merge_to_the_unsplit_result(device, code, hq, hkv, d, world, context, partition, broken):
    """Records of every rank's pages, merged. A row that is not finite reaches the result of its heads through both merges."""
    import torch

    from khalamari_b200 import abi, split_kv
    from khalamari_b200.device import Buffer, Dtype
    full = _full(code, hq, hkv, d, context)
    records, keep = [], []
    for rank, (begin, end) in enumerate(split_kv.split_context(context, world, full.page)):
        run = ScaledRun(device, _local(full, begin, end, 100 + rank, broken), max_tokens=256)
        decode = split_kv.SplitKvDecode(device, run.attention, 1)
        decode.prepare(run.case.slots[0], end - begin, partition)
        decode.record_local(run.stream, run.q, run.pages, run.ids)
        run.stream.synchronize()
        torch.cuda.synchronize()
        assert device.check(run.stream) == 0
        records.append(decode.local_record.clone())
        keep.append((run, decode))
    gathered = torch.cat(records)
    torch.cuda.synchronize()
    run = keep[0][0]
    out = Buffer.new_zeroed(device, hq * d * 2)
    abi.call("kh_combine_packed_partials", device.handle, run.stream.handle, world, hq, d,
             Buffer.wrap(device, gathered.data_ptr(), gathered.numel() * 4).ref, int(Dtype.Bfloat16), out.ref)
    run.stream.synchronize()
    _check(bits_to_f32("bf16", out.read(0, hq * d, np.uint16)).reshape(1, hq, d), full, broken)


@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("world,my_rank,broken", [(1, 0, None), (4, 2, None), (1, 0, (1000, 1)), (4, 2, (1600, 0)), (4, 2, (10, 1))])
def test_peer_exchange_over_scaled_pages(device, code, world, my_rank, broken):
    """The one-kernel exchange: (1600, 0) is a row of this rank, (10, 1) one whose NaN another rank delivers."""
    from khalamari_b200 import split_kv
    from khalamari_b200.device import Buffer
    hq, hkv, d, context = 16, 2, 128, 3000
    full = _full(code, hq, hkv, d, context)
    ranges = split_kv.split_context(context, world, full.page)
    q = bits_to_f32("bf16", full.q_bits)[0].astype(np.float64)
    record, step = d + 4, 1
    image = np.zeros(2 * world * hq * record, np.float32)
    flags = np.zeros(2 * world * hq + hq, np.uint32)
    for rank, (begin, end) in enumerate(ranges):
        if rank == my_rank:
            continue
        for h in range(hq):
            head = h // (hq // hkv)
            s = full.k[0][begin:end, head] @ q[h] * full.scale
            p = np.exp(s - s.max())
            at = (((step & 1) * world + rank) * hq + h) * record
            image[at:at + d] = p @ full.v[0][begin:end, head] / p.sum()
            image[at + d], image[at + d + 1] = p.sum(), s.max()
            if broken is not None and begin <= broken[0] < end and head == broken[1]:
                image[at:at + d + 1] = np.nan  # as the exchange kernel delivers it: NaN, under a finite maximum
                image[at + d + 1] = 0.0
            flags[((step & 1) * world + rank) * hq + h] = step
    exchange = split_kv.PeerExchange(device, my_rank, world, hq, d)
    exchange.inbox.write(0, np.concatenate([image.view(np.uint32), flags]))
    scratch = [Buffer.new_zeroed(device, exchange.inbox.len_bytes()) for _ in range(world)]
    exchange.attach([exchange.inbox.ref.ptr if r == my_rank else scratch[r].ref.ptr for r in range(world)])
    begin, end = ranges[my_rank]
    run = ScaledRun(device, _local(full, begin, end, 300, broken), max_tokens=256)
    decode = split_kv.SplitKvDecode(device, run.attention, world, peer_exchange=exchange)
    decode.prepare(run.case.slots[0], end - begin, 128)
    out = Buffer.new_zeroed(device, hq * d * 2)
    decode.record_step(run.stream, run.q, run.pages, run.ids, out)
    run.stream.synchronize()
    assert device.check(run.stream) == 0
    _check(bits_to_f32("bf16", out.read(0, hq * d, np.uint16)).reshape(1, hq, d), full, broken)
    exchange.close()


@pytest.mark.parametrize("code", CODES)
def test_a_step_of_one_rank_keeps_nan(device, code):
    """record_step: map, local merge, merge of the gathered records."""
    import torch

    from khalamari_b200 import split_kv
    from khalamari_b200.device import Buffer, Stream
    hq, hkv, d, context = 16, 2, 128, 2000
    full = _full(code, hq, hkv, d, context)
    stream = Stream(device, torch.cuda.current_stream().cuda_stream)
    run = ScaledRun(device, _local(full, 0, context, 5, (700, 1)), max_tokens=256)
    decode = split_kv.SplitKvDecode(device, run.attention, 1)
    decode.prepare(run.case.slots[0], context, 256)
    out = Buffer.new_zeroed(device, hq * d * 2)
    decode.record_step(stream, run.q, run.pages, run.ids, out)
    torch.cuda.synchronize()
    assert device.check(stream) == 0
    _check(bits_to_f32("bf16", out.read(0, hq * d, np.uint16)).reshape(1, hq, d), full, (700, 1))
