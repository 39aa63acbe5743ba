"""Workloads of the scaled 8-bit KV cache: quantising page write, page read-back and attention over such pages.

A cache page holds, for every KV head, K and V rows of ``head_dim`` 8-bit codes and one scale byte per row:
``[K/V][Hkv][P][D]`` codes, then ``[Hkv][K/V][P]`` scale bytes ``b``. A row stands for ``code * 2^(b - 127)`` (``b`` = 0: a
row of zeros; 255: not finite). Codes are int8 or FP8 E4M3FN. With ``own`` false the operators are computed in plain torch
operations in 32 bits; with ``own`` true through this package's entry points.
"""
import random

import torch

own = False

IO = {"bf16": torch.bfloat16, "f16": torch.float16}


# ---- cases ------------------------------------------------------------------------------------------------------
def _cache(op, code, io, hkv, d, page, **more):
    return {"op": op, "code": code, "io": io, "hkv": hkv, "d": d, "page": page, **more}


def _attend(code, io, hq, hkv, d, page, batch, q_len, low, high, lengths):
    return _cache("attend", code, io, hkv, d, page, hq=hq, batch=batch, q_len=q_len, low=low, high=high, lengths=lengths)


def listed():
    cases = {
        # the new rows of one decode step of four sequences: latency of the two launches
        "round trip 4 rows": _cache("round_trip", "int8", "f16", 2, 256, 16, batch=4, q_len=1),
        # one decode step of 64 sequences
        "round trip 64 rows": _cache("round_trip", "e4m3", "bf16", 8, 128, 16, batch=64, q_len=1),
        # eight prefill chunks of 2,048 tokens
        "round trip 16384 rows": _cache("round_trip", "int8", "bf16", 8, 128, 16, batch=8, q_len=2048),
        # four contexts read back whole (cache export, swap-out)
        "read 117k rows": _cache("read", "int8", "bf16", 4, 256, 16, batch=4, q_len=29333),
        # ragged medium read of 8-token pages
        "read 3k rows": _cache("read", "e4m3", "f16", 8, 128, 8, batch=3, q_len=1021),
        # four short sequences, one new token each: latency
        "decode 4": _attend("int8", "f16", 16, 2, 256, 16, 4, 1, 128, 2048, 0),
        # 64 sequences, 32 layers' worth of them make a decode step: HBM-bound
        "decode 64": _attend("int8", "bf16", 64, 8, 128, 16, 64, 1, 1024, 8192, 1),
        "decode 64 e4m3": _attend("e4m3", "bf16", 64, 8, 128, 16, 64, 1, 1024, 8192, 1),
        # speculative verify: one token and three drafts over long prefixes
        "verify 32": _attend("int8", "bf16", 24, 4, 256, 16, 32, 4, 4096, 32768, 2),
        # one very long sequence
        "decode 1 long": _attend("int8", "bf16", 16, 2, 256, 16, 1, 1, 524288, 524288, 3),
        # chunked prefill: causal chunks behind ragged prefixes
        "prefill 4": _attend("int8", "bf16", 64, 8, 128, 16, 4, 2048, 2048, 12288, 4),
        # a short prompt, odd length, head_dim 256
        "prefill 1 short": _attend("e4m3", "f16", 16, 2, 256, 32, 1, 517, 517, 517, 5),
    }
    return [dict(case, name=name) for name, case in cases.items()]


def _spread(rng, low, high):
    return int(round(low * (high / low) ** rng.random()))


def draw(rng):
    d = rng.choice((128, 256))
    page = rng.choice((8, 16, 16, 16) if d == 128 else (8, 16, 16, 32))
    hkv = rng.choice((1, 2, 4, 8) if d == 128 else (1, 2, 4))
    code, io = rng.choice(("int8", "e4m3")), rng.choice(("bf16", "f16"))
    kind = rng.choice(("round_trip", "read", "decode", "decode", "verify", "prefill"))
    if kind == "round_trip":
        batch = _spread(rng, 1, 64)
        return _cache(kind, code, io, hkv, d, page, batch=batch, q_len=_spread(rng, 1, 16384 // batch))
    if kind == "read":
        batch = _spread(rng, 1, 16)
        return _cache(kind, code, io, hkv, d, page, batch=batch, q_len=_spread(rng, 1, 65536 // batch))
    hq = hkv * rng.choice((1, 2, 4, 5, 6, 7, 8))
    lengths = rng.randrange(1 << 20)
    if kind == "decode":
        batch = _spread(rng, 1, 96)
        high = _spread(rng, 16, min(65536, 400000 // batch))
        return _attend(code, io, hq, hkv, d, page, batch, 1, max(1, high // rng.choice((1, 2, 8))), high, lengths)
    if kind == "verify":
        batch, q_len = _spread(rng, 1, 32), rng.choice((2, 3, 4, 5, 8))
        high = _spread(rng, 64, min(32768, 400000 // batch))
        return _attend(code, io, hq, hkv, d, page, batch, q_len, max(q_len, high // 4), high, lengths)
    batch = rng.choice((1, 2, 3, 4))
    q_len = _spread(rng, 16, 2048)
    high = _spread(rng, q_len, 12288)
    return _attend(code, io, hq, hkv, d, page, batch, q_len, q_len, high, lengths)


def _contexts(case):
    """Tokens in the cache for each sequence, the new ones among them."""
    if case["op"] != "attend":
        return [case["q_len"]] * case["batch"]
    rng = random.Random(case["lengths"])
    return [rng.randint(case["low"], case["high"]) for _ in range(case["batch"])]


def work(case):
    hkv, d, q = case["hkv"], case["d"], case["q_len"]
    row8, row16 = 2 * hkv * (d + 1), 2 * hkv * d * 2
    if case["op"] != "attend":
        rows = case["batch"] * q
        if case["op"] == "read":
            return {"bytes": rows * (row8 + row16), "flops": rows * 2 * hkv * d}
        return {"bytes": 2 * rows * (row8 + row16), "flops": rows * 2 * hkv * d * 4}
    contexts = _contexts(case)
    pairs = sum(q * c - q * (q - 1) // 2 for c in contexts)
    return {"bytes": sum(contexts) * row8 + 2 * len(contexts) * q * case["hq"] * d * 2,
            "flops": 4 * case["hq"] * d * pairs}


# ---- the operators in plain torch operations ----------------------------------------------------------------------
def _power(b):
    """2^(b - 127) of a scale byte, 0 for 0, NaN for 255."""
    power = (b.int() << 23).view(torch.float32)
    return torch.where(b == 255, torch.full_like(power, float("nan")), power)


def _quantise(x, code):
    """Rows of 32-bit values to (codes as bytes, scale bytes)."""
    top = x.abs().amax(-1)
    fraction, exponent = torch.frexp(top)  # top = fraction * 2^exponent, fraction in [1/2, 1)
    if code == "int8":  # top * 2^-e < 127.5
        b = exponent - 7 + (fraction >= 127.5 / 128).int() + 127
    else:  # top * 2^-e <= 448
        b = exponent - 9 + (fraction > 448 / 512).int() + 127
    b = torch.where(top > 0, b.clamp(min=1), torch.zeros_like(b))
    y = x * ((254 - b).int() << 23).view(torch.float32).unsqueeze(-1)
    codes = torch.round(y).to(torch.int8) if code == "int8" else y.to(torch.float8_e4m3fn)
    return codes.view(torch.uint8), b.to(torch.uint8)


def _values(codes, b, code):
    kind = torch.int8 if code == "int8" else torch.float8_e4m3fn
    return codes.view(kind).float() * _power(b).unsqueeze(-1)


def _planes(case, pool):
    """Views of the pool: codes [pages][2][Hkv][P][D] and scale bytes [pages][Hkv][2][P]."""
    hkv, d, page = case["hkv"], case["d"], case["page"]
    split = 2 * hkv * page * d
    return (pool[:, :split].unflatten(1, (2, hkv, page, d)), pool[:, split:].unflatten(1, (hkv, 2, page)))


def _write(case, s):
    codes, scales = _planes(case, s["pool"])
    page = s["page_ids"][s["slots"].long(), s["tokens"].long() // case["page"]].long()
    at = s["tokens"].long() % case["page"]
    for plane, rows in enumerate((s["k"], s["v"])):
        c, b = _quantise(rows.float(), case["code"])
        codes[page, plane, :, at] = c
        scales[page, :, plane, at] = b


def _read(case, s):
    codes, scales = _planes(case, s["pool"])
    page = s["page_ids"][s["slots"].long(), s["tokens"].long() // case["page"]].long()
    at = s["tokens"].long() % case["page"]
    most = torch.finfo(IO[case["io"]]).max
    return [_values(codes[page, plane, :, at], scales[page, :, plane, at], case["code"]).clamp(-most, most).to(IO[case["io"]])
            for plane in (0, 1)]


def _gather(case, s, plane):
    """[batch][Hkv][longest][D] values of K or V, zero rows past a sequence's end."""
    codes, scales = _planes(case, s["pool"])
    ids = s["page_ids"].long()
    x = _values(codes[ids, plane], scales[ids, :, plane], case["code"])  # [batch][pages][Hkv][P][D]
    return x.transpose(1, 2).flatten(2, 3)[:, :, :s["longest"]]


def _attention(case, s):
    batch, q_len, d, hkv = case["batch"], case["q_len"], case["d"], case["hkv"]
    group = case["hq"] // hkv
    q = s["q"].float().view(batch, q_len, hkv, group, d).permute(0, 2, 3, 1, 4).reshape(batch, hkv, group * q_len, d)
    scores = (q * d ** -0.5) @ _gather(case, s, 0).transpose(-1, -2)
    scores = scores.view(batch, hkv, group, q_len, -1)
    t = torch.arange(s["longest"], device=q.device)
    last = s["contexts"].view(-1, 1) - q_len + torch.arange(q_len, device=q.device)
    hidden = t > last.unsqueeze(-1)
    scores.masked_fill_(hidden.view(batch, 1, 1, q_len, -1), float("-inf"))
    scores.sub_(scores.amax(-1, keepdim=True)).exp_()
    total = scores.sum(-1, keepdim=True)
    v = _gather(case, s, 1)
    out = (scores.view(batch, hkv, group * q_len, -1) @ v).view(batch, hkv, group, q_len, d) / total
    return out.permute(0, 3, 1, 2, 4).reshape(batch * q_len, case["hq"], d).to(IO[case["io"]])


# ---- inputs -------------------------------------------------------------------------------------------------------
def _fresh_rows(case, rows, generator):
    """K and V rows as a layer makes them: a few K channels are several times larger, V rows differ in size."""
    shape = (rows, case["hkv"], case["d"])
    k = torch.randn(shape, generator=generator, device="cuda")
    channel = torch.rand((1, case["hkv"], case["d"]), generator=generator, device="cuda")
    k *= torch.where(channel < 0.03, 5.0, 1.0)
    v = torch.randn(shape, generator=generator, device="cuda")
    v *= torch.exp(0.5 * torch.randn((rows, 1, 1), generator=generator, device="cuda"))
    return k.to(IO[case["io"]]), v.to(IO[case["io"]])


def prepare(case, seed):
    generator = torch.Generator("cuda").manual_seed(seed)
    page, hkv, d, batch, q_len = case["page"], case["hkv"], case["d"], case["batch"], case["q_len"]
    contexts = _contexts(case)
    blocks = max(-(-c // page) for c in contexts)
    pages = batch * blocks
    page_ids = torch.randperm(pages, generator=generator, device="cuda").to(torch.int32).view(batch, blocks)
    s = {"case": case, "contexts": torch.tensor(contexts, device="cuda"), "longest": max(contexts), "page_ids": page_ids,
         "pool": torch.zeros(pages, 2 * hkv * page * (d + 1), dtype=torch.uint8, device="cuda")}
    if case["op"] == "round_trip":
        s["k"], s["v"] = _fresh_rows(case, batch * q_len, generator)
    else:
        codes, scales = _planes(case, s["pool"])
        per = max(1, (1 << 27) // (hkv * page * d))
        for first in range(0, pages, per):  # the cache as earlier steps left it, some pages at a time
            n = min(per, pages - first)
            for plane, rows in enumerate(_fresh_rows(case, n * page, generator)):
                c, b = _quantise(rows.float(), case["code"])
                codes[first:first + n, plane] = c.view(n, page, hkv, d).transpose(1, 2)
                scales[first:first + n, :, plane] = b.view(n, page, hkv).transpose(1, 2)
    if case["op"] == "attend":
        s["q"] = torch.randn((batch * q_len, case["hq"], d), generator=generator, device="cuda").to(IO[case["io"]])
        s["out"] = torch.empty_like(s["q"])
    else:
        s["slots"] = torch.arange(batch, device="cuda", dtype=torch.int32).repeat_interleave(q_len)
        s["tokens"] = torch.arange(q_len, device="cuda", dtype=torch.int32).repeat(batch)
        s["k_out"] = torch.empty((batch * q_len, hkv, d), dtype=IO[case["io"]], device="cuda")
        s["v_out"] = torch.empty_like(s["k_out"])
    if own:
        s["plan"] = _plan(case, s, contexts)
    return s


# ---- the same through this package ----------------------------------------------------------------------------------
_device = None


def _plan(case, s, contexts):
    """What a serving program keeps: the device and stream handles, the components, the batch's plan."""
    global _device
    from khalamari_b200 import kv_page_read, kv_page_write
    from khalamari_b200.device import Buffer, Device, Dtype, Stream
    from khalamari_b200.gqa import GQAAttention, GQACore
    from khalamari_b200.request_page_table import GQAPageTableLayout

    if _device is None:
        _device = Device(torch.cuda.current_device())
    io = Dtype.Bfloat16 if case["io"] == "bf16" else Dtype.Float16
    kv = Dtype.Int8Scaled if case["code"] == "int8" else Dtype.Fp8E4M3Scaled
    batch, blocks = s["page_ids"].shape
    layout = GQAPageTableLayout(batch, 1, blocks, 1)

    def buffer(name):
        return Buffer.wrap(_device, s[name].data_ptr(), s[name].numel() * s[name].element_size())

    plan = {"stream": Stream(_device, torch.cuda.current_stream().cuda_stream)}
    page_bytes = s["pool"].shape[1]
    if case["op"] == "attend":
        core = GQACore(case["d"], case["hq"], case["hkv"], case["d"] ** -0.5)
        tokens = batch * case["q_len"]
        plan["attention"] = GQAAttention(_device, core, io, page_bytes, layout, tokens, kv_dtype=kv)
        plan["attention"].prepare(list(range(batch)), [c - case["q_len"] for c in contexts],
                                  [r * case["q_len"] for r in range(batch + 1)], tokens)
        plan["buffers"] = [buffer(name) for name in ("q", "pool", "page_ids", "out")]
        return plan
    rows = s["tokens"].numel()
    if case["op"] == "round_trip":
        plan["write"] = kv_page_write.Compute(_device, kv_page_write.Config(case["hkv"], case["d"], page_bytes, io, kv))
        plan["write_shape"] = kv_page_write.Shape(rows, layout)
        plan["write_buffers"] = kv_page_write.Buffers(*map(buffer, ("pool", "k", "v", "slots", "tokens", "page_ids")))
    plan["read"] = kv_page_read.Compute(_device, kv_page_read.Config(case["hkv"], case["d"], page_bytes, io, kv))
    plan["read_shape"] = kv_page_read.Shape(rows, layout)
    plan["read_buffers"] = kv_page_read.Buffers(*map(buffer, ("pool", "k_out", "v_out", "slots", "tokens", "page_ids")))
    return plan


def run(s):
    case = s["case"]
    if own:
        plan = s["plan"]
        if case["op"] == "attend":
            plan["attention"].record_sdpa(plan["stream"], *plan["buffers"])
            return s["out"]
        rows = s["tokens"].numel()
        if case["op"] == "round_trip":
            plan["write"].invoke(plan["stream"], plan["write_shape"], plan["write_buffers"], rows)
        plan["read"].invoke(plan["stream"], plan["read_shape"], plan["read_buffers"], rows)
        return [s["k_out"], s["v_out"]]
    if case["op"] == "attend":
        return _attention(case, s)
    if case["op"] == "round_trip":
        _write(case, s)
    return _read(case, s)


# ---- the definition in 64 bits ----------------------------------------------------------------------------------------
def _two(n):
    """2^n in 64 bits, from the format's exponent field."""
    return ((n.to(torch.int64) + 1023) << 52).view(torch.float64)


def _decode64(raw, byte, code):
    """Values of code bytes [..., D] under scale bytes [...], from the formats' definitions."""
    raw = raw.to(torch.int64)
    if code == "int8":
        value = torch.where(raw > 127, raw - 256, raw).double()
    else:
        field, mantissa = (raw >> 3) & 15, (raw & 7).double()
        size = torch.where(field == 0, mantissa / 512, (1 + mantissa / 8) * _two(field - 7))
        value = torch.where(raw > 127, -size, size)
    power = _two(byte.to(torch.int64) - 127)
    return value * torch.where(byte == 0, torch.zeros_like(power), power).unsqueeze(-1)


def _round64(x, code):
    """What a row of 64-bit values becomes in the cache: the smallest power of two that fits it, codes to the nearest even."""
    top = x.abs().amax(-1, keepdim=True)
    low = torch.floor(torch.log2(torch.where(top > 0, top, torch.ones_like(top)))) - 9
    for _ in range(5):
        y = top * _two(-low)
        low = torch.where((torch.round(y) > 127) if code == "int8" else (y > 448), low + 1, low)
    low = low.clamp(min=-126)
    y = x * _two(-low)
    if code != "int8":
        size = torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6)))
        size = torch.where(y.abs() < _two(size), size - 1, size).clamp(min=-6)
        step = _two(size - 3)
        return torch.round(y / step) * step * _two(low)
    return torch.round(y) * _two(low)


def exact(case, seed):
    s = prepare(case, seed)
    page, hkv, d, q_len = case["page"], case["hkv"], case["d"], case["q_len"]
    if case["op"] == "round_trip":
        return [_round64(s[name].double(), case["code"]) for name in ("k", "v")]
    split = 2 * hkv * page * d
    codes = s["pool"][:, :split].reshape(-1, 2, hkv, page, d)
    scales = s["pool"][:, split:].reshape(-1, hkv, 2, page)

    def rows(r, plane, head, n):
        ids = s["page_ids"][r].long()
        return _decode64(codes[ids, plane, head].reshape(-1, d)[:n], scales[ids, head, plane].reshape(-1)[:n], case["code"])

    if case["op"] == "read":
        return [torch.cat([torch.stack([rows(r, plane, h, q_len) for h in range(hkv)], 1) for r in range(case["batch"])])
                for plane in (0, 1)]
    group = case["hq"] // hkv
    out = torch.empty(s["q"].shape, dtype=torch.float64, device="cuda")
    for r, context in enumerate(s["contexts"].tolist()):
        q = s["q"][r * q_len:(r + 1) * q_len].double()
        seen = torch.arange(context, device="cuda") <= (context - q_len + torch.arange(q_len, device="cuda")).view(-1, 1)
        for h in range(hkv):
            k, v = rows(r, 0, h, context), rows(r, 1, h, context)
            for j in range(h * group, (h + 1) * group):
                logits = (q[:, j] @ k.T) / d ** 0.5
                weight = torch.softmax(logits.masked_fill(~seen, float("-inf")), -1)
                out[r * q_len:(r + 1) * q_len, j] = weight @ v
    return out
