"""GPU parity of the paged key/value cache (append with rotary embedding, reading back, attention) against oracle/kv.py in 64 bits.

Bars, written down before the first run.  A rounding to type t is off by eps_t / 2 of the value (fp16 2^-11, bf16 2^-8, fp32 2^-24).
  append, 16 bits: fp32 products of a 16-bit value with a cosine and a sine rounded to fp32, their sum rounded to fp32 (4 roundings
    at most on |a| + |b|), then one rounding to the type; values are copied bit for bit.
  append, codes: equal codes (the rotated key is 64-bit up to its code), scales to one rounding to fp32 plus one of their quotient.
  attention: scores are fp32 sums of exact products: relative to sum |q k| off by d + 4 roundings, taken twice as large (2^-23) since
    the tensor cores may cut instead of rounding; a probability off by twice that, by exp2 in fp32 (2^-21) and by its rounding for the
    second product (fp16 2^-11 plus 2^-25 of the largest, bf16 2^-8); the sum over the keys another 2^-22 a key; the result eps / 2.
"""
import numpy as np
import pytest

from oracle import kv as okv
from tests.gpu_util import from_bf16_bits, gpu, to_bf16_bits  # noqa: F401

pytestmark = pytest.mark.gpu

F16, BF16, F32 = 9, 12, 10
HALF_STEP = {F16: 2.0 ** -11, BF16: 2.0 ** -8, F32: 2.0 ** -24}


def raw(x, dtype):
    """The 16-bit patterns of values."""
    return np.asarray(x, np.float16).view(np.uint16) if dtype == F16 else to_bf16_bits(np.asarray(x, np.float32))


def values(bits, dtype):
    return (bits.view(np.float16) if dtype == F16 else from_bf16_bits(bits)).astype(np.float64)


def random_rows(rng, shape, dtype, factor=1.0):
    return raw(rng.standard_normal(shape) * factor, dtype)


class Setup:
    """A pool, the sequences [(new, length), ...] over shuffled pages, and the same in numpy.  Everything that no row may see is poison."""

    def __init__(self, seqs, dtype=F16, bits=16, kv_heads=2, head_dim=128, page=16, seed=0, gap=0, tail=3, window=0, spare=2):
        from mlxl3_b200 import kv
        from mlxl3_b200.runtime import DeviceBuffer
        self.kv, self.Buffer = kv, DeviceBuffer
        self.seqs, self.dtype, self.bits, self.kv_heads, self.d, self.page = seqs, dtype, bits, kv_heads, head_dim, page
        rng = self.rng = np.random.default_rng([seed, 77])
        self.start = gap + np.concatenate(([0], np.cumsum([n for n, _ in seqs])))
        self.rows = int(self.start[-1]) + tail
        self.width = max(1, max(-(-length // page) for _, length in seqs)) + 1
        used = sum(-(-length // page) for _, length in seqs)
        self.pages = used + spare
        order = rng.permutation(self.pages)
        self.table = np.full((len(seqs), self.width), -1, np.int32)
        at = 0
        for b, (_, length) in enumerate(seqs):
            c = -(-length // page)
            self.table[b, :c] = order[at:at + c]
            at += c
        shape = (self.pages, kv_heads, page)
        nan = raw(np.full(1, np.nan), dtype)[0]
        self.pool, self.scale = {}, {}
        for name in "kv":
            if bits == 16:
                self.pool[name] = np.full(shape + (head_dim,), nan, np.uint16)
            else:
                self.pool[name] = rng.integers(0, 256, shape + (head_dim * bits // 8,), dtype=np.uint8)
                self.scale[name] = np.full(shape, np.nan, np.float32)
        # tokens that some row sees
        for b, (n, length) in enumerate(seqs):
            first = max(0, length - n + 1 - window) if window else 0
            for t in range(first, length if n else 0):
                at = self.table[b, t // page], slice(None), t % page
                for name in "kv":
                    x = rng.standard_normal((kv_heads, head_dim)) * (1.0 if name == "k" else rng.uniform(0.5, 2.0))
                    if bits == 16:
                        self.pool[name][at] = raw(x, dtype)
                    else:
                        codes, scale = okv.quantise(x, bits)
                        self.pool[name][at], self.scale[name][at] = okv.pack(codes, bits), scale
        self.upload()

    def upload(self):
        up = self.Buffer.from_numpy
        self.dev = {name: up(self.pool[name]) for name in "kv"}
        self.dev_scale = {name: up(s) for name, s in self.scale.items()}
        self.d_start, self.d_length = up(self.start.astype(np.int32)), up(np.array([length for _, length in self.seqs], np.int32))
        self.d_table = up(self.table)
        self.cache = self.kv.KvCache(self.pages, self.page, self.kv_heads, self.d, self.dtype, self.bits, self.dev["k"].ptr, self.dev["v"].ptr,
                                     *(self.dev_scale[n].ptr if self.bits != 16 else 0 for n in "kv"))
        self.batch = self.kv.KvBatch(self.d_start.ptr, self.d_length.ptr, self.d_table.ptr, len(self.seqs), self.width, self.rows)

    def held(self, name, b, t):
        """What the pool holds for tokens t of sequence b, in 64 bits."""
        t = np.asarray(t)
        at = self.table[b, t // self.page], slice(None), t % self.page
        if self.bits == 16:
            return values(self.pool[name][at], self.dtype)
        return okv.unpack(self.pool[name][at], self.bits) * self.scale[name][at].astype(np.float64)[..., None]

    def download(self):
        pool = {n: self.dev[n].download(self.pool[n].shape, self.pool[n].dtype) for n in "kv"}
        return pool, {n: self.dev_scale[n].download(self.scale[n].shape, np.float32) for n in self.scale}


# ---- append -----------------------------------------------------------------------------------------------------------


def run_append(s, heads, rotated, interleaved, magnitude, theta=10000.0, wide=0, in_place=False):
    up, rng, d = s.Buffer.from_numpy, s.rng, s.d
    turns = s.kv.rope_turns(rotated, theta) if rotated else np.zeros(0)
    d_turns = up(turns if rotated else np.zeros(2))
    rope = s.kv.Rope(d_turns.ptr, rotated, interleaved, magnitude)
    width = heads * d + 2 * s.kv_heads * d + wide
    qkv = random_rows(rng, (s.rows, width), s.dtype)
    d_qkv = up(qkv)
    sentinel = raw(np.full((s.rows, heads * d), 7.0), s.dtype)
    d_out = up(sentinel)
    k_at, v_at = heads * d * 2, (heads + s.kv_heads) * d * 2
    s.kv.append(s.cache, s.batch, d_qkv.ptr + k_at, d_qkv.ptr + v_at, rope, d_q=d_qkv.ptr if heads else 0, heads=heads,
                d_q_out=(d_qkv.ptr if in_place else d_out.ptr) if heads else 0, q_stride=width if heads else 0,
                q_out_stride=width if in_place else 0, k_stride=width, v_stride=width)
    if in_place:
        got = d_qkv.download(qkv.shape, np.uint16)
        assert np.array_equal(got[:, heads * d:], qkv[:, heads * d:])
        return turns, qkv, got[:, :heads * d], qkv[:, :heads * d]
    return turns, qkv, d_out.download(sentinel.shape, np.uint16), sentinel


def check_append(s, heads, rotated, interleaved, magnitude, result):
    turns, qkv, got_q, untouched = result
    d, g = s.d, s.kv_heads
    x = values(qkv, s.dtype)
    pool, scale = s.download()
    want_pool, want_scale = {n: s.pool[n].copy() for n in "kv"}, {n: v.copy() for n, v in s.scale.items()}
    bound_step, live = HALF_STEP[s.dtype], np.zeros(s.rows, bool)

    def close(got, row, position):
        want = okv.rope(row, position, turns, interleaved, magnitude)
        parts = np.abs(row)
        if rotated:
            pairs = (np.abs(row[..., 0:rotated:2]) + np.abs(row[..., 1:rotated:2])).repeat(2, -1) if interleaved else \
                np.tile(np.abs(row[..., :rotated // 2]) + np.abs(row[..., rotated // 2:rotated]), 2)
            parts = np.concatenate((pairs * abs(magnitude), parts[..., rotated:]), -1)
        inner = 4 * 2.0 ** -24 * parts * (np.arange(d) < rotated)
        tolerance = bound_step * (np.abs(want) + inner) + inner + (2.0 ** -25 if s.dtype == F16 else 0.0)
        assert (np.abs(values(got, s.dtype) - want) <= tolerance).all()
    for b, (n, length) in enumerate(s.seqs):
        for i in range(n):
            row, position = int(s.start[b]) + i, length - n + i
            if position < 0:
                continue
            live[row] = True
            if heads:
                close(got_q[row].reshape(heads, d), x[row, :heads * d].reshape(heads, d), position)
            k = x[row, heads * d:(heads + g) * d].reshape(g, d)
            v = x[row, (heads + g) * d:(heads + 2 * g) * d].reshape(g, d)
            page = s.table[b, position // s.page] if position // s.page < s.width else -1
            if not 0 <= page < s.pages:
                continue
            at = page, slice(None), position % s.page
            if s.bits == 16:
                close(pool["k"][at], k, position)
                want_pool["k"][at] = pool["k"][at]
                want_pool["v"][at] = raw(v, s.dtype)
            else:
                for name, vec in (("k", okv.rope(k, position, turns, interleaved, magnitude)), ("v", v)):
                    codes, sc = okv.quantise(vec, s.bits)
                    want_pool[name][at] = okv.pack(codes, s.bits)
                    assert (np.abs(scale[name][at].astype(np.float64) - sc) <= 2.0 ** -23 * np.abs(sc)).all()
                    want_scale[name][at] = scale[name][at]
    for n in "kv":
        assert np.array_equal(pool[n], want_pool[n])                              # equal codes, and nothing else was written
        if s.bits != 16:
            assert np.array_equal(scale[n].view(np.uint32), want_scale[n].view(np.uint32))
    assert np.array_equal(got_q[~live], untouched[~live])


SEQS = [(1, 1), (5, 5), (0, 9), (3, 40), (17, 130), (4, 2), (2, 0)]


@pytest.mark.parametrize("bits", [16, 8, 4])
@pytest.mark.parametrize("dtype,d,rotated,interleaved,page,heads", [
    (F16, 128, 128, False, 16, 8), (BF16, 128, 64, True, 32, 6), (F16, 64, 64, True, 24, 3), (BF16, 64, 16, False, 7, 4), (F16, 128, 48, False, 64, 2),
    (BF16, 128, 0, False, 1, 2), (F16, 64, 32, True, 256, 0)])
def test_append(gpu, bits, dtype, d, rotated, interleaved, page, heads):
    s = Setup(SEQS, dtype, bits, kv_heads=2 if heads != 3 else 3, head_dim=d, page=page, seed=bits + rotated, gap=2)
    check_append(s, heads, rotated, interleaved, 1.25, run_append(s, heads, rotated, interleaved, 1.25, wide=8))


@pytest.mark.parametrize("bits", [16, 4])
def test_append_many_rows_in_place(gpu, bits):
    # more rows than a CTA each is started for
    s = Setup([(900, 900), (1, 70), (410, 500)], F16, bits, kv_heads=1, head_dim=64, page=32, seed=3, gap=1)
    check_append(s, 2, 64, False, 1.0, run_append(s, 2, 64, False, 1.0, in_place=True))


def test_append_far_positions_and_batches_beyond_shared_memory(gpu):
    # one page is enough for rows far behind: the table names it for every index
    s = Setup([(1, 3)] * 300, BF16, 8, kv_heads=1, head_dim=64, page=16, seed=4)
    check_append(s, 1, 64, True, 1.0, run_append(s, 1, 64, True, 1.0))
    far = Setup([(2, 40)], F16, 8, kv_heads=1, head_dim=128, page=16, seed=5)
    length = 1 << 24
    far.seqs, far.width = [(2, length)], length // 16
    far.table = np.full((1, far.width), 1, np.int32)
    far.upload()
    check_append(far, 1, 128, False, 1.0, run_append(far, 1, 128, False, 1.0, theta=500000.0))


def test_append_values_that_are_not_finite_or_zero(gpu):
    s = Setup([(4, 4)], F16, 8, kv_heads=1, head_dim=64, page=16, tail=0)
    up = s.Buffer.from_numpy
    x = np.ones((4, 64), np.float16)
    x[0], x[1, 3], x[2, 5] = 0.0, np.nan, np.inf
    d = up(x)
    s.kv.append(s.cache, s.batch, d.ptr, d.ptr)
    out = [s.Buffer(4 * 64 * 4) for _ in range(2)]
    s.kv.read(s.cache, s.batch, F32, out[0].ptr, out[1].ptr)
    for o in out:
        got = o.download((4, 64), np.float32)
        assert (got[0] == 0).all() and np.isnan(got[1:3]).all() and np.abs(got[3] - 1).max() <= 2.0 ** -23


def test_append_and_read_outside_table_and_pool(gpu):
    s = Setup([(40, 40), (3, 20)], F16, 16, kv_heads=2, head_dim=64, page=16)
    s.table[0, 1] = s.pages                  # tokens 16..31: no such page
    s.table[1, 1] = -5
    s.width = 2                              # and the table ends before token 32
    s.table = np.ascontiguousarray(s.table[:, :2])
    s.upload()
    check_append(s, 2, 64, False, 1.0, run_append(s, 2, 64, False, 1.0))
    pool, _ = s.download()
    sentinel = np.full((s.rows, 2, 64), 5.0, np.float32)
    out = [s.Buffer.from_numpy(sentinel) for _ in range(2)]
    s.kv.read(s.cache, s.batch, F32, out[0].ptr, out[1].ptr)
    for name, o in zip("kv", out):
        got = o.download(sentinel.shape, np.float32)
        want = sentinel.copy()
        want[:16] = values(pool[name][s.table[0, 0], :, :16].transpose(1, 0, 2).copy(), F16)
        assert np.array_equal(got, want)
    # lengths and first rows that make no sense stay inside the buffers
    for start, length in (([0, 1 << 30, -7], [1 << 31 - 1, -4]), ([-9, -3, 1 << 30], [40, 40]), ([43, 3, 0], [20, 20])):
        s.d_start.upload(np.array(start, np.int64).astype(np.int32))
        s.d_length.upload(np.array(length, np.int64).astype(np.int32))
        run_append(s, 2, 64, False, 1.0)
        s.kv.read(s.cache, s.batch, F32, out[0].ptr, out[1].ptr)
        ws = s.kv.new_attention_workspace(s.cache, s.batch, 2)
        s.kv.attention(s.cache, s.batch, out[0].ptr, 2, 0.1, out[1].ptr, ws)
        out[0].download(sentinel.shape, np.float32)


# ---- read -------------------------------------------------------------------------------------------------------------


@pytest.mark.parametrize("out", [F16, BF16, F32])
@pytest.mark.parametrize("dtype,bits,d,page", [(F16, 16, 128, 16), (BF16, 16, 64, 5), (F16, 8, 64, 32), (BF16, 8, 128, 16), (F16, 4, 128, 64), (BF16, 4, 64, 24)])
def test_read(gpu, out, dtype, bits, d, page):
    seqs = [(1, 1), (33, 33), (0, 5), (7, 130), (3, 1)] + ([(2800, 2900)] if d == 64 else [])
    s = Setup(seqs, dtype, bits, kv_heads=2, head_dim=d, page=page, seed=out, gap=1)
    size = 4 if out == F32 else 2
    sentinel = np.full(s.rows * 2 * d * size, 0x3c, np.uint8)
    bufs = [s.Buffer.from_numpy(sentinel) for _ in range(2)]
    s.kv.read(s.cache, s.batch, out, bufs[0].ptr, bufs[1].ptr)
    for name, buf in zip("kv", bufs):
        got = buf.download((s.rows, 2, d), np.float32 if size == 4 else np.uint16)
        live = np.zeros(s.rows, bool)
        for b, (n, length) in enumerate(s.seqs):
            for i in range(max(0, n - length), n):
                row = int(s.start[b]) + i
                live[row] = True
                want = s.held(name, b, [length - n + i])[0]
                have = got[row].astype(np.float64) if out == F32 else values(got[row], out)
                tolerance = HALF_STEP[out] * np.abs(want) * (1 + 2.0 ** -20) + (2.0 ** -24 * np.abs(want)) + (2.0 ** -25 if out == F16 else 0.0)
                assert (np.abs(have - want) <= tolerance).all()
        assert (got[~live].view(np.uint8) == 0x3c).all()
    # one output alone
    again = s.Buffer.from_numpy(sentinel)
    s.kv.read(s.cache, s.batch, out, 0, again.ptr)
    assert np.array_equal(again.download(sentinel.shape, np.uint8), bufs[1].download(sentinel.shape, np.uint8))


# ---- attention --------------------------------------------------------------------------------------------------------


def attend(s, heads, window=0, max_new=0, q_factor=1.5, wide=0, workspace=None, stream=None):
    from mlxl3_b200.runtime import DEFAULT_STREAM
    width = heads * s.d + wide
    q = random_rows(s.rng, (s.rows, width), s.dtype, q_factor)
    sentinel = raw(np.full((s.rows, width), 9.0), s.dtype)
    d_q, d_out = s.Buffer.from_numpy(q), s.Buffer.from_numpy(sentinel)
    workspace = workspace or s.kv.new_attention_workspace(s.cache, s.batch, heads, max_new)
    scale = s.d ** -0.5

    def call():
        s.kv.attention(s.cache, s.batch, d_q.ptr, heads, scale, d_out.ptr, workspace, max_new, window, width, width, stream or DEFAULT_STREAM)
        return d_out.download(sentinel.shape, np.uint16, stream or DEFAULT_STREAM)
    got = call()
    check_attention(s, heads, q, got, sentinel, window, max_new)
    assert np.array_equal(got, call())                                        # parts are joined in a fixed order
    header = workspace.download((16384,), np.uint8, stream or DEFAULT_STREAM)
    assert not header.any()
    return got


def check_attention(s, heads, q, got, untouched, window=0, max_new=0):
    d, scale = s.d, s.d ** -0.5
    product = s.dtype if s.bits == 16 else F16
    live = np.zeros(got.shape, bool)
    worst = 0.0
    for b, (n, length) in enumerate(s.seqs):
        use = min(n, max_new) if max_new else n
        if not use:
            continue
        rows = slice(int(s.start[b]), int(s.start[b]) + use)
        low = max(0, length - n + 1 - window) if window else 0
        keys, vals = (np.zeros((length, s.kv_heads, d)) for _ in range(2))
        if length > low:
            keys[low:], vals[low:] = s.held("k", b, np.arange(low, length)), s.held("v", b, np.arange(low, length))
        qv = values(q[rows, :heads * d], s.dtype).reshape(use, heads, d)
        want, mass, most, seen, top_v = okv.attention(qv, keys, vals, length - n, scale, window)
        live[rows, :heads * d] = True
        score = (d + 4) * 2.0 ** -23 * most
        if s.bits != 16:
            # rows in fp16 after a power of two: 2^-25 of the row's largest, over the keys' vectors
            score = score + scale * 2.0 ** -24 * np.abs(qv).max(-1) * (np.abs(keys).sum(-1).max() if length > low else 0.0)
        small = 2.0 ** -25 * seen * top_v if product == F16 else 0.0 * seen
        relative = np.expm1(2 * score) + 2.0 ** -20 + HALF_STEP[product] + seen * 2.0 ** -22
        tolerance = (relative * 1.0)[..., None] * mass + small[..., None]
        tolerance = tolerance + HALF_STEP[s.dtype] * (np.abs(want) + tolerance) + (2.0 ** -25 if s.dtype == F16 else 0.0)
        error = np.abs(values(got[rows, :heads * d], s.dtype).reshape(use, heads, d) - want)
        assert np.isfinite(error).all()
        worst = max(worst, float((error / np.maximum(tolerance, 1e-30)).max()))
    assert worst <= 1.0, f"{worst} of the bound"
    assert np.array_equal(got[~live], untouched[~live])


DECODE = [(1, 1), (1, 64), (1, 65), (0, 30), (1, 200), (1, 700), (1, 0)]
CHUNKS = [(3, 3), (1, 130), (0, 0), (40, 41), (70, 300), (5, 2), (2, 500)]


@pytest.mark.parametrize("bits", [16, 8, 4])
@pytest.mark.parametrize("dtype,d,heads,kv_heads,page", [(F16, 128, 8, 2, 16), (BF16, 128, 5, 1, 64), (F16, 64, 14, 2, 24), (BF16, 64, 3, 3, 1), (BF16, 128, 16, 1, 128),
                                                         (F16, 128, 40, 2, 32)])
def test_attention_single_tokens(gpu, bits, dtype, d, heads, kv_heads, page):
    s = Setup(DECODE, dtype, bits, kv_heads, d, page, seed=heads + bits)
    attend(s, heads, max_new=1)


@pytest.mark.parametrize("bits", [16, 8, 4])
@pytest.mark.parametrize("dtype,d,heads,kv_heads,page,window", [(F16, 128, 8, 2, 16, 0), (BF16, 128, 5, 1, 64, 100), (F16, 64, 14, 2, 24, 0), (BF16, 64, 3, 3, 50, 33),
                                                                (F16, 128, 2, 2, 256, 1)])
def test_attention_chunks(gpu, bits, dtype, d, heads, kv_heads, page, window):
    s = Setup(CHUNKS, dtype, bits, kv_heads, d, page, seed=heads + bits + 100, window=window, gap=1)
    attend(s, heads, window, wide=16)


@pytest.mark.parametrize("new,heads,kv_heads", [(4, 8, 2), (5, 8, 2), (16, 4, 2), (33, 2, 2), (16, 5, 1)])
def test_attention_few_rows_per_key_head(gpu, new, heads, kv_heads):
    # on both sides of the row counts at which another kernel takes over
    s = Setup([(new, 300), (1, 90), (new, new)], BF16, 16, kv_heads, 128, 16, seed=new)
    attend(s, heads, max_new=new)


@pytest.mark.parametrize("bits", [16, 8])
def test_attention_long(gpu, bits):
    # one sequence over many CTAs; one that ends inside the first block of a page
    s = Setup([(1, 6001), (1, 17)], F16, bits, 1, 64, 16, seed=bits)
    attend(s, 4, max_new=1)


@pytest.mark.parametrize("bits", [16, 8, 4])
@pytest.mark.parametrize("dtype,d,heads,kv_heads,page,window,seqs", [
    (F16, 128, 4, 1, 16, 0, [(700, 700), (1, 90), (130, 900), (0, 4), (33, 40)]), (BF16, 128, 2, 2, 64, 0, [(257, 1500)]),
    (BF16, 64, 14, 2, 24, 200, [(300, 300), (20, 777)]), (F16, 64, 2, 2, 128, 0, [(128, 128), (129, 129), (256, 511)]),
    (F16, 128, 5, 1, 32, 64, [(16, 1200), (26, 26), (200, 150)]), (BF16, 128, 8, 8, 16, 0, [(300, 2000)])])
def test_attention_prompts(gpu, bits, dtype, d, heads, kv_heads, page, window, seqs):
    s = Setup(seqs, dtype, bits, kv_heads, d, page, seed=heads + bits + 200, window=window, gap=3)
    attend(s, heads, window, wide=8)


def test_attention_maximum_that_climbs(gpu):
    # every key scores higher than the ones before, by far more than a row's maximum is left behind
    s = Setup([(140, 1000)], F16, 16, 1, 128, 16, seed=30)
    one = np.ones(128) / 8
    for t in range(1000):
        s.pool["k"][s.table[0, t // 16], 0, t % 16] = raw(one * (t / 40.0), F16)
    s.upload()
    width, heads = 2 * 128, 2
    q = raw(np.ones((s.rows, width)) * 2.0, F16)
    d_q, d_out = s.Buffer.from_numpy(q), s.Buffer.from_numpy(q)
    ws = s.kv.new_attention_workspace(s.cache, s.batch, heads)
    s.kv.attention(s.cache, s.batch, d_q.ptr, heads, 128 ** -0.5, d_out.ptr, ws)
    check_attention(s, heads, q, d_out.download(q.shape, np.uint16), q)


def test_attention_rows_beyond_max_new(gpu):
    s = Setup([(6, 90), (2, 40)], F16, 16, 2, 128, 16, seed=8)
    attend(s, 4, max_new=3)


def test_attention_scales_of_any_magnitude(gpu):
    # quantised keys and values far from one: the largest of the type, and so small that fp16 could not hold a product
    for k_size, v_size in ((1e-3, 1e-6), (40.0, 3e4)):
        s = Setup([(1, 150), (3, 70)], BF16, 8, 1, 64, 16, seed=9)
        for name, size in (("k", k_size), ("v", v_size)):
            s.scale[name] = s.scale[name] * np.float32(size)
        s.upload()
        attend(s, 4, q_factor=1.0 / k_size)


@pytest.mark.parametrize("bits", [16, 4])
def test_attention_more_sequences_than_shared_memory_names(gpu, bits):
    rng = np.random.default_rng(31)
    few = Setup([(1, int(n)) for n in rng.integers(1, 40, 150)], F16, bits, 1, 64, 16, seed=31)
    attend(few, 2, max_new=1)
    many = Setup([(int(n), int(n) + 3) for n in rng.integers(0, 6, 530)], BF16, bits, 1, 64, 16, seed=32)
    attend(many, 4, max_new=6)


@pytest.mark.parametrize("bits", [8, 4])
def test_scales_that_bulk_copies_cannot_read(gpu, bits):
    # scale arrays that lie on 4 bytes only: every key goes the slow way
    s = Setup([(1, 200), (30, 170)], F16, bits, 2, 128, 32, seed=33)
    for name in "kv":
        buf = s.Buffer(s.scale[name].nbytes + 16)
        buf.upload(s.scale[name], offset=4)
        s.dev_scale[name] = buf
    s.cache = s.kv.KvCache(s.pages, s.page, s.kv_heads, s.d, s.dtype, s.bits, s.dev["k"].ptr, s.dev["v"].ptr, *(s.dev_scale[n].ptr + 4 for n in "kv"))
    attend(s, 4)
    attend(s, 4, max_new=2)


def test_attention_pages_outside_the_pool_read_as_zeros(gpu):
    for bits in (16, 8):
        s = Setup([(1, 100), (40, 90)], F16, bits, 1, 64, 16, seed=34, spare=2)
        held = s.held
        s.table[0, 2], s.table[1, 1] = s.pages + 5, -7
        s.upload()

        def zeros_there(name, b, t):
            t = np.asarray(t)
            x, bad = np.zeros((len(t), 1, 64)), (t // 16 == 2) if b == 0 else (t // 16 == 1)
            x[~bad] = held(name, b, t[~bad])
            return x
        s.held = zeros_there
        attend(s, 4, max_new=40)
        s.seqs = s.seqs[:1]
        s.batch = s.kv.KvBatch(s.d_start.ptr, s.d_length.ptr, s.d_table.ptr, 1, s.width, s.rows)
        attend(s, 4, max_new=1)


def test_attention_shares_a_workspace_and_streams(gpu):
    from mlxl3_b200.runtime import Stream
    a = Setup([(1, 900)], F16, 16, 2, 128, 16, seed=10)
    b = Setup([(37, 200), (1, 333)], BF16, 4, 1, 64, 32, seed=11)
    ws = a.kv.new_attention_workspace(a.cache, b.batch, 8, 64)
    for _ in range(2):                                                        # calls of different shapes one after the other
        attend(a, 8, max_new=1, workspace=ws)
        attend(b, 2, workspace=ws)
    attend(a, 8, max_new=1, stream=Stream())


def test_step_recorded_and_replayed_while_sequences_grow(gpu):
    """append -> attention of one token per step, recorded once; the lengths advance on the device between replays."""
    from mlxl3_b200.runtime import Graph, Stream
    heads, steps = 4, 5
    s = Setup([(1, 40), (1, 1), (1, 129)], F16, 16, 2, 64, 16, seed=12, tail=0, spare=8)
    free = [p for p in range(s.pages) if p not in set(s.table[s.table >= 0].tolist())]
    for b, (_, length) in enumerate(s.seqs):
        if (length + steps) // 16 > (length - 1) // 16:
            s.table[b, (length - 1) // 16 + 1] = free.pop()
    s.upload()
    up, stream, d = s.Buffer.from_numpy, Stream(), s.d
    turns = s.kv.rope_turns(64, 10000.0)
    d_turns = up(turns)
    rope = s.kv.Rope(d_turns.ptr, 64)
    qkv = s.Buffer(3 * (heads + 4) * d * 2)
    out = s.Buffer(3 * heads * d * 2)
    ws = s.kv.new_attention_workspace(s.cache, s.batch, heads, 1)
    width = (heads + 4) * d

    def launch():
        s.kv.append(s.cache, s.batch, qkv.ptr + heads * d * 2, qkv.ptr + (heads + 2) * d * 2, rope, qkv.ptr, heads, qkv.ptr, width, width, width, width, stream)
        s.kv.attention(s.cache, s.batch, qkv.ptr, heads, d ** -0.5, out.ptr, ws, 1, 0, width, 0, stream)
    first = random_rows(s.rng, (3, width), F16)
    qkv.upload(first, stream)
    launch()
    stream.sync()
    with Graph.record(stream) as graph:
        launch()
    for step in range(steps):
        s.seqs = [(1, length + (1 if step else 0)) for _, length in s.seqs]
        x = random_rows(s.rng, (3, width), F16)
        qkv.upload(x, stream)
        s.d_length.upload(np.array([length for _, length in s.seqs], np.int32), stream)
        graph.launch(stream)
        rotated = qkv.download((3, width), np.uint16, stream)
        s.pool, _ = s.download()
        for b, (_, length) in enumerate(s.seqs):
            k = okv.rope(values(x[b], F16)[heads * d:(heads + 2) * d].reshape(2, d), length - 1, turns)
            assert np.abs(s.held("k", b, [length - 1])[0] - k).max() <= 2.0 ** -10 * 8
        got = out.download((3, heads * d), np.uint16, stream)
        check_attention(s, heads, rotated[:, :heads * d], got, got)


@pytest.mark.parametrize("bits", [16, 8, 4])
def test_prompt_in_pieces_equals_prompt_at_once(gpu, bits):
    """A prompt of 150 tokens appended and attended in pieces of 1, 60 and 89 against the same at once."""
    heads, kv_heads, d, total = 4, 2, 128, 150
    rng = np.random.default_rng(13)
    width = (heads + 2 * kv_heads) * d
    qkv = random_rows(rng, (total, width), F16)
    outs = []
    for pieces in ([150], [1, 60, 89]):
        s = Setup([(total, total)], F16, bits, kv_heads, d, 16, seed=14, tail=0)
        up = s.Buffer.from_numpy
        d_turns, d_x, d_out = up(s.kv.rope_turns(128, 10000.0)), up(qkv), s.Buffer(total * heads * d * 2)
        rope, done = s.kv.Rope(d_turns.ptr, 128), 0
        for n in pieces:
            d_start, d_length = up(np.array([0, n], np.int32)), up(np.array([done + n], np.int32))
            batch = s.kv.KvBatch(d_start.ptr, d_length.ptr, s.d_table.ptr, 1, s.width, n)
            at = d_x.ptr + done * width * 2
            s.kv.append(s.cache, batch, at + heads * d * 2, at + (heads + kv_heads) * d * 2, rope, at, heads, at, width, width, width, width)
            ws = s.kv.new_attention_workspace(s.cache, batch, heads)
            s.kv.attention(s.cache, batch, at, heads, d ** -0.5, d_out.ptr + done * heads * d * 2, ws, q_stride=width)
            done += n
        rotated = d_x.download(qkv.shape, np.uint16)
        s.pool, s.scale = s.download()
        got = d_out.download((total, heads * d), np.uint16)
        check_attention(s, heads, rotated[:, :heads * d], got, got)
        outs.append((rotated, s.pool["k"], s.pool["v"]))
    for a, b in zip(*outs):
        assert np.array_equal(a, b)


def test_decoder_prefill_equals_steps(gpu):
    """A prompt through ``DenseDecoder.prefill`` (in one piece, and in two) against the same tokens one step at a time, and the step after it.
    Bar: that of a decode step in tests/test_gpu_decoder.py, 3e-2 of the largest logit."""
    from mlxl3_b200.decoder import DecoderConfig, DenseDecoder, SyntheticWeights
    config = DecoderConfig(layers=2, hidden=512, heads=4, kv_heads=2, head_dim=128, ffn=1024, vocab=1024, k_bits=4, codebook=0, max_ctx=48)
    weights = SyntheticWeights(config, seed=11)
    tokens = np.random.default_rng(5).integers(0, 1024, 24).astype(np.int32)
    steps = DenseDecoder(config, weights)
    steps.store_logits = True
    for i, token in enumerate(tokens):
        steps.set_input(int(token), i)
        steps.step()
    want = steps.download("logits").astype(np.float32)
    for pieces in ((24,), (1, 23), (17, 7)):
        model = DenseDecoder(config, weights)
        model.store_logits = True
        done = 0
        for n in pieces:
            model.prefill(tokens[done:done + n], done)
            done += n
        got = model.download("logits").astype(np.float32)
        assert np.abs(got - want).max() <= 3e-2 * np.abs(want).max()
        assert want[model.result()[1]] >= want.max() - 3e-2 * np.abs(want).max()
        for d in (model, steps):
            d.set_input(7, 24)
            d.step()
        after, after_want = (d.download("logits").astype(np.float32) for d in (model, steps))
        assert np.abs(after - after_want).max() <= 3e-2 * np.abs(after_want).max()
    with pytest.raises(gpu.B200Exl3Error, match="do not fit"):
        model.prefill(tokens, 30)


@pytest.mark.parametrize("pdl", [0, 1, 2])
def test_chain_of_calls_with_and_without_dependent_launch(gpu, pdl):
    """append -> attention -> append of the outputs -> read, back to back, for a mixed batch: the same bits whether kernels start early or not."""
    import mlxl3_b200
    results = []
    for option in (0, pdl):
        s = Setup([(1, 300), (40, 400), (2, 5), (100, 100)], BF16, 8, 2, 64, 16, seed=40, tail=0)
        up, heads, d = s.Buffer.from_numpy, 4, s.d
        width = (heads + 4) * d
        qkv = up(random_rows(np.random.default_rng(41), (s.rows, width), BF16))
        turns = up(s.kv.rope_turns(64, 10000.0))
        rope = s.kv.Rope(turns.ptr, 64, True)
        out, k, v = s.Buffer(s.rows * heads * d * 2), s.Buffer(s.rows * 2 * d * 4), s.Buffer(s.rows * 2 * d * 4)
        ws = s.kv.new_attention_workspace(s.cache, s.batch, heads)
        mlxl3_b200.set_option("pdl", option)
        try:
            for _ in range(3):
                s.kv.append(s.cache, s.batch, qkv.ptr + heads * d * 2, qkv.ptr + (heads + 2) * d * 2, rope, qkv.ptr, heads, qkv.ptr, width, width, width, width)
                s.kv.attention(s.cache, s.batch, qkv.ptr, heads, 0.125, out.ptr, ws, q_stride=width)
                s.kv.append(s.cache, s.batch, out.ptr, out.ptr + 2 * d * 2, k_stride=heads * d, v_stride=heads * d)
                s.kv.read(s.cache, s.batch, F32, k.ptr, v.ptr)
            results.append([b.download((b.nbytes,), np.uint8) for b in (qkv, out, k, v)])
        finally:
            mlxl3_b200.set_option("pdl", 0)
    for a, b in zip(*results):
        assert np.array_equal(a, b)
