"""Plain 64-bit restatement of the scaled 8-bit cache (codes and one power-of-two scale byte per token and KV head),
seeded cases over it, and the runner that takes them through the package's entry points."""
from __future__ import annotations

import math
from dataclasses import dataclass

import numpy as np

from helpers import bits_to_f32, nan_bits, round_to

CODES = ("int8", "e4m3")


def e4m3_table() -> np.ndarray:
    """Value of every E4M3FN code, from the format's definition."""
    code = np.arange(256)
    field, mantissa = (code >> 3) & 15, (code & 7).astype(np.float64)
    size = np.where(field == 0, mantissa / 512, (1 + mantissa / 8) * np.exp2(field - 7.0))
    size[(code & 127) == 127] = np.nan
    return np.where(code > 127, -size, size)


E4M3 = e4m3_table()


def quantise(values: np.ndarray, code: str) -> tuple[np.ndarray, np.ndarray]:
    """Rows [..., D] to (code bytes, scale bytes): the smallest exponent e >= -126 whose scaled row rounds into the
    codes' range; codes to nearest, ties to even. Finite rows only."""
    x = np.asarray(values, dtype=np.float64)
    top = np.abs(x).max(-1)
    # start below any answer and raise while the largest value does not fit
    e = np.where(top > 0, np.floor(np.log2(np.where(top > 0, top, 1.0))) - 10, 0).astype(np.int64)
    for _ in range(8):
        y = top * np.exp2(-e.astype(np.float64))
        e += (np.rint(y) > 127) if code == "int8" else (y > 448)
    e = np.maximum(e, -126)
    y = x * np.exp2(-e.astype(np.float64))[..., None]
    if code == "int8":
        codes = np.rint(y).astype(np.int64) & 255
    else:
        _, exponent = np.frexp(np.abs(y))
        step = np.exp2(np.maximum(exponent - 1, -6) - 3.0)
        rounded = np.rint(y / step) * step
        order = np.argsort(E4M3[:127])
        codes = order[np.searchsorted(E4M3[:127][order], np.abs(rounded))]
        assert np.array_equal(E4M3[codes], np.abs(rounded))
        codes = codes + 128 * np.signbit(y)
    b = np.where(top > 0, e + 127, 0)
    codes = np.where((top > 0)[..., None], codes, 0)
    return codes.astype(np.uint8), b.astype(np.uint8)


def values_of(codes: np.ndarray, scale: np.ndarray, code: str) -> np.ndarray:
    raw = codes.astype(np.int8).astype(np.float64) if code == "int8" else E4M3[codes]
    power = np.where(scale == 0, 0.0, np.exp2(scale.astype(np.float64) - 127))
    power[scale == 255] = np.nan
    return raw * power[..., None]


def page_bytes(hkv: int, page: int, d: int) -> int:
    return 2 * hkv * page * (d + 1)


def planes(pool: np.ndarray, hkv: int, page: int, d: int) -> tuple[np.ndarray, np.ndarray]:
    """Views of a byte pool: codes [pages, 2, Hkv, P, D] and scale bytes [pages, Hkv, 2, P]."""
    pages = pool.reshape(-1, page_bytes(hkv, page, d))
    split = 2 * hkv * page * d
    return pages[:, :split].reshape(-1, 2, hkv, page, d), pages[:, split:].reshape(-1, hkv, 2, page)


@dataclass
class ScaledCase:
    code: str
    dtype_name: str
    hq: int
    hkv: int
    d: int
    page: int
    scale: float
    histories: list
    q_lens: list
    slots: list
    q_bits: np.ndarray
    pool: np.ndarray
    table: np.ndarray   # [slots][layers][blocks][ids per block]
    layer: int
    k: list             # per request [context, Hkv, D] values the cache stands for
    v: list

    @property
    def cu(self) -> list:
        return [0] + np.cumsum(self.q_lens).tolist()

    def visible(self) -> list:
        """Per flat Q token (request, begin, end): causal."""
        return [(r, 0, h + i + 1) for r, (h, n) in enumerate(zip(self.histories, self.q_lens)) for i in range(n)]


def make_scaled_case(seed, code, dtype_name, hq, hkv, d, histories, q_lens, page=16, layers=1, layer=0, ids_per_block=1,
                     k_scale=None, v_scale=None, poison=0xFF, scale=None) -> ScaledCase:
    """Cache rows drawn as normal values times ``k_scale`` / ``v_scale`` ([token, head] magnitudes), quantised here;
    the rest of the pool holds ``poison`` (0xff: NaN codes and NaN scale bytes)."""
    rng = np.random.default_rng(seed)
    contexts = [h + n for h, n in zip(histories, q_lens)]
    needed = [-(-c // page) for c in contexts]
    blocks = -(-max(needed) // ids_per_block)
    num_slots = len(contexts) + 1
    slots = rng.permutation(num_slots)[:len(contexts)].tolist()
    total = sum(needed)
    pool = np.full((total + 3) * page_bytes(hkv, page, d), poison, np.uint8)
    codes, scales = planes(pool, hkv, page, d)
    free = rng.permutation(total + 3)
    table = np.full((num_slots, layers, blocks * ids_per_block), 0xFFFFFFFF, np.uint32)  # unallocated entries: garbage
    ks, vs, used = [], [], 0
    for r, context in enumerate(contexts):
        ids = free[used:used + needed[r]]
        used += needed[r]
        table[slots[r], layer, :needed[r]] = ids
        at, row = ids[np.arange(context) // page], np.arange(context) % page
        for plane, (out, factor) in enumerate(((ks, k_scale), (vs, v_scale))):
            x = rng.standard_normal((context, hkv, d))
            if factor is not None:
                x *= factor(rng, context, hkv)[..., None]
            _, x = round_to(dtype_name, x.astype(np.float32))
            c, b = quantise(x, code)
            codes[at, plane, :, row] = c
            scales[at, :, plane, row] = b
            out.append(values_of(c, b, code))
    q_bits, _ = round_to(dtype_name, rng.standard_normal((sum(q_lens), hq, d)).astype(np.float32))
    return ScaledCase(code, dtype_name, hq, hkv, d, page, scale or d ** -0.5, list(histories), list(q_lens), slots, q_bits,
                      pool, table, layer, ks, vs)


def reference(case: ScaledCase, visible=None, wide: bool = False) -> tuple[np.ndarray, np.ndarray]:
    """(attention output, per-element error bound) in 64 bits.

    The bound counts what the kernels round: the output, half a step of its type; the value weights, to f16 (half a
    step: 2^-11 of each term; 2^-8 where a ``wide`` Q tile, of more than 32 rows (24 at head_dim 256), has
    bf16 probabilities), plus 2^-25 of the largest weight where a weight is subnormal there - references lie at
    most 2^8 below the largest weight, and a code is at most twice the row's largest code, so 2^-25 * 2 * largest
    |p v| per token); and f32 arithmetic on the scores: a dot product of D terms is off by at most D * 2^-23 of the
    sum of magnitudes (additions that may truncate), a handful of roundings of the score and of exp2 add 2^-20 of
    the largest score magnitude and 2^-20: the probabilities are off by that, relatively, twice (numerator and sum)."""
    q = bits_to_f32(case.dtype_name, case.q_bits).reshape(-1, case.hq, case.d).astype(np.float64)
    group = case.hq // case.hkv
    out, bound = np.zeros_like(q), np.zeros_like(q)
    eps = 2.0 ** -8 if case.dtype_name == "bf16" else 2.0 ** -11
    tiny = 0.0 if case.dtype_name == "bf16" else 2.0 ** -25
    for token, (r, begin, end) in enumerate(visible if visible is not None else case.visible()):
        if end <= begin:
            continue
        k, v = case.k[r][begin:end], case.v[r][begin:end]
        for head in range(case.hq):
            kh, vh = k[:, head // group], v[:, head // group]
            s = (kh @ q[token, head]) * case.scale
            p = np.exp(s - s.max())
            p /= p.sum()
            o = p @ vh
            size = p @ np.abs(vh)
            dot = case.scale * (np.abs(kh) @ np.abs(q[token, head])).max()
            relative = (2.0 ** -8 if wide and case.dtype_name == "bf16" else 2.0 ** -11) + 2 * (case.d * 2.0 ** -23 * dot + 2.0 ** -20 * (1 + np.abs(s).max() * 1.5))
            floor = len(p) * 2.0 ** -24 * (p[:, None] * np.abs(vh)).max()
            out[token, head] = o
            bound[token, head] = eps * np.abs(o) + tiny + 1.01 * (relative * size + floor)
    return out, bound


def assert_close(actual, expected, bound, what=""):
    actual = np.asarray(actual, np.float64)
    assert np.all(np.isfinite(actual)), f"{what}: non-finite output"
    error = np.abs(actual - expected)
    assert np.all(error <= bound), f"{what}: worst error is {float((error / np.maximum(bound, 1e-300)).max()):.3f} bounds"


class ScaledRun:
    """A ``ScaledCase`` on the device, through ``GQAAttention``."""

    def __init__(self, device, case: ScaledCase, max_tokens=None, policy=None, selector=None):
        from khalamari_b200.device import Buffer, Dtype, Stream
        from khalamari_b200.gqa import GQAAttention, GQACore
        from khalamari_b200.request_page_table import GQAPageTableLayout
        from khalamari_b200.selector import SelectorPolicy

        self.case, self.device = case, device
        self.io = Dtype.Bfloat16 if case.dtype_name == "bf16" else Dtype.Float16
        self.kv = Dtype.Int8Scaled if case.code == "int8" else Dtype.Fp8E4M3Scaled
        slots, layers, ids = case.table.shape
        self.layout = GQAPageTableLayout(slots, layers, ids, 1)
        self.stream = Stream(device)
        self.pages = Buffer.from_slice(device, case.pool)
        self.ids = Buffer.from_slice(device, case.table.reshape(-1))
        tokens = len(case.q_bits)
        self.attention = GQAAttention(device, GQACore(case.d, case.hq, case.hkv, case.scale), self.io,
                                      page_bytes(case.hkv, case.page, case.d), self.layout, max_tokens or tokens,
                                      SelectorPolicy.B200 if policy is None else policy, selector, kv_dtype=self.kv)
        self.row = case.hq * case.d
        capacity = self.attention.policy.q_token_ranges.capacity(tokens)
        q = np.full(capacity * self.row, nan_bits(case.dtype_name), np.uint16)
        q[:tokens * self.row] = case.q_bits.reshape(-1)
        self.q = Buffer.from_slice(device, q)
        self.canary = 0x4228
        self.out_rows = capacity + 2
        self.out = Buffer.from_slice(device, np.full(self.out_rows * self.row, self.canary, np.uint16))

    def plan(self, selection=None):
        case = self.case
        return self.attention.prepare(case.slots, case.histories, case.cu, selection=selection)

    def record(self):
        self.attention.record_sdpa(self.stream, self.q, self.pages, self.ids, self.out, self.case.layer)

    def wide(self) -> bool:
        block = self.attention.metadata.variant().thread_block
        return block.max_q_tokens * block.max_q_heads > (32 if self.case.d == 128 else 24)

    def read(self):
        self.stream.synchronize()
        assert self.device.check(self.stream) == 0
        tokens = len(self.case.q_bits)
        bits = self.out.read(0, self.out_rows * self.row, np.uint16)
        assert np.all(bits[tokens * self.row:] == self.canary), "rows past the active tokens were written"
        return bits_to_f32(self.case.dtype_name, bits[:tokens * self.row]).reshape(tokens, self.case.hq, self.case.d)

    def run(self, selection=None):
        self.plan(selection)
        self.record()
        return self.read()
