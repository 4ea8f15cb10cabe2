"""GPU tests of the paged key/value cache at the ends of its ranges: magnitudes of keys, values and scales, windows and lengths, numbers that
are not finite where a row must not see them.  The bars are those of tests/test_gpu_kv.py, with the terms that a test adds written beside it.
"""
import numpy as np
import pytest

from oracle import kv as okv
from tests.gpu_util import gpu  # noqa: F401
from tests.test_gpu_kv import BF16, F16, F32, HALF_STEP, Setup, raw, values  # noqa: F401

pytestmark = pytest.mark.gpu


def run_attention(s, heads, q, window=0, max_new=0):
    """Outputs [rows, heads, d] in 64 bits; the same bits twice, and a clean workspace header."""
    d_q, d_out = s.Buffer.from_numpy(q), s.Buffer.from_numpy(q)
    ws = s.kv.new_attention_workspace(s.cache, s.batch, heads, max_new)
    got = []
    for _ in range(2):
        s.kv.attention(s.cache, s.batch, d_q.ptr, heads, s.d ** -0.5, d_out.ptr, ws, max_new, window)
        got.append(d_out.download(q.shape, np.uint16))
    assert np.array_equal(*got) and not ws.download((16384,), np.uint8).any()
    return values(got[0], s.dtype).reshape(s.rows, heads, s.d)


def largest_term(s, qv, keys, vals, first_position, scale):
    """Largest probability times largest |value| of a key, [rows, heads]."""
    n, heads, _ = qv.shape
    group, out = heads // s.kv_heads, np.zeros((n, heads))
    for i in range(n):
        end = first_position + i + 1
        for h in range(heads if end > 0 else 0):
            x = scale * (keys[:end, h // group] @ qv[i, h])
            p = np.exp(x - x.max())
            out[i, h] = (p / p.sum() * np.abs(vals[:end, h // group]).max(-1)).max()
    return out


def rows_want(s, heads, q, b, window=0, by_term=False):
    """(rows, what they should hold, the bar, visible keys) of sequence b.  by_term: fp16 products hold a term, the probability times the
    value, to 2^-11 of itself or, subnormal, to 2^-25 in a unit of which the row's largest term makes 2^7 at least."""
    n, length = s.seqs[b]
    rows = slice(int(s.start[b]), int(s.start[b]) + n)
    low = max(0, length - n + 1 - window) if window else 0
    keys, vals = (np.zeros((length, s.kv_heads, s.d)) for _ in range(2))
    keys[low:], vals[low:] = s.held("k", b, np.arange(low, length)), s.held("v", b, np.arange(low, length))
    qv = values(q[rows], s.dtype).reshape(n, heads, s.d)
    want, mass, most, seen, top_v = okv.attention(qv, keys, vals, length - n, s.d ** -0.5, window)
    score = (s.d + 4) * 2.0 ** -23 * most
    if s.bits != 16:
        score = score + s.d ** -0.5 * 2.0 ** -24 * np.abs(qv).max(-1) * np.abs(keys).sum(-1).max(initial=0.0)
    product = s.dtype if s.bits == 16 else F16
    bar = (np.expm1(2 * score) + 2.0 ** -20 + HALF_STEP[product] + seen * 2.0 ** -22)[..., None] * mass
    small = 2.0 ** -32 * largest_term(s, qv, keys, vals, length - n, s.d ** -0.5) if by_term else 2.0 ** -25 * top_v
    bar = bar + (seen * small if product == F16 else 0.0 * seen)[..., None]
    bar = bar + HALF_STEP[s.dtype] * (np.abs(want) + bar) + (2.0 ** -25 if s.dtype == F16 else 0.0)
    return rows, want, bar, seen


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("size", [1e-39, 1e-45])
@pytest.mark.parametrize("new", [1, 3, 40])
def test_value_scales_without_an_inverse(gpu, bits, size, new):
    """Scales of the smallest numbers of fp32, some of them zero: over a whole sequence, and ahead of ordinary tokens.  A value scale is held
    to 2^-96 or better (scales below 2^-100 are as good as zero), times the largest code, for each key."""
    s = Setup([(new, 130), (new, 40 + new), (new, 300)], BF16, bits, 1, 64, 16, seed=50 + new, tail=0)
    for b, last in ((0, 130), (1, 40 + new), (2, 70)):
        t = np.arange(last)
        at = s.table[b, t // 16], 0, t % 16
        s.scale["v"][at] = np.where(t % 3 == 1, 0.0, size).astype(np.float32)
        if b == 1:
            s.scale["k"][at] = np.where(t % 5 == 1, 0.0, s.scale["k"][at])
    s.upload()
    q = raw(s.rng.standard_normal((s.rows, 2 * 64)), BF16)
    got = run_attention(s, 2, q, max_new=new)
    for b in range(3):
        rows, want, bar, seen = rows_want(s, 2, q, b)
        assert (np.abs(got[rows] - want) <= bar + (seen * okv.LIMIT[bits] * 2.0 ** -96)[..., None]).all()


@pytest.mark.parametrize("bits", [8, 4])
def test_codes_of_the_largest_values(gpu, bits):
    """bf16 vectors up to the largest number of the type, half of the largest (a middle between two codes: the even one) among them: equal codes."""
    rng = np.random.default_rng(51)
    s = Setup([(64, 64)], BF16, bits, 1, 128, 16, seed=51, tail=0)
    x = rng.standard_normal((64, 128)) * 2.0 ** rng.integers(96, 126, (64, 1))
    top = (1.0 + rng.integers(0, 128, 64) / 128.0) * 2.0 ** rng.integers(96, 128, 64)
    x = np.clip(x, -top[:, None], top[:, None])
    x[:, 3], x[:, 7], x[:, 11] = top, top / 2, -top / 2
    x[0, 3:12] = 2.0 ** 127, 2.0 ** 126, -2.0 ** 126, 2.0 ** 125, 1.5 * 2.0 ** 126, 0.0, 1.0, 2.0 ** 119, 2.0 ** 120
    stored = raw(x, BF16)
    x = values(stored, BF16)
    assert np.isfinite(x).all()
    d_x = s.Buffer.from_numpy(stored)
    s.kv.append(s.cache, s.batch, d_x.ptr, d_x.ptr)
    pool, scale = s.download()
    codes, want_scale = okv.quantise(x, bits)
    t = np.arange(64)
    at = s.table[0, t // 16], 0, t % 16
    for name in "kv":
        assert np.array_equal(okv.unpack(pool[name][at], bits), codes)
        assert (np.abs(scale[name][at].astype(np.float64) - want_scale) <= 2.0 ** -23 * want_scale).all()


@pytest.mark.parametrize("bits", [16, 8])
@pytest.mark.parametrize("seqs", [[(8, 3), (1, 5)], [(40, 30), (130, 4), (2, 0)]])
def test_windows_beyond_every_length(gpu, bits, seqs):
    """A window of the largest int hides nothing, also for rows ahead of their sequence's first token."""
    s = Setup(seqs, F16, bits, 1, 64, 16, seed=52, tail=0)
    q = raw(s.rng.standard_normal((s.rows, 2 * 64)), F16)
    open_end = run_attention(s, 2, q)
    for window in (2 ** 31 - 1, 2 ** 30, 200):
        assert np.array_equal(run_attention(s, 2, q, window), open_end)
    for b in range(len(seqs)):
        rows, want, bar, seen = rows_want(s, 2, q, b)
        assert (np.abs(open_end[rows] - want) <= bar).all()


def test_second_tile_waits_through_a_long_run(gpu):
    """Half a second of sequences of one tile, every CTA's run without a break, and behind them one of two tiles: its second tile's rows have
    waited since the call began.  The long ones share a page of equal tokens: every output is their value."""
    from mlxl3_b200 import kv
    from mlxl3_b200.runtime import DeviceBuffer
    length, long_ones, rows, d = 1 << 20, 6400, 33, 64
    last = Setup([(70, 300)], F16, 8, 1, d, 512, seed=53, tail=0)
    ends = []                                            # the last sequence's page lies behind the long ones' in pools of its own
    for name in "kv":
        pool, scale = DeviceBuffer(2 * length * d), DeviceBuffer.from_numpy(np.ones(2 * length, np.float32))
        pool.fill(1)
        pool.upload(last.pool[name][last.table[0, 0], 0], offset=length * d)
        scale.upload(last.scale[name][last.table[0, 0], 0], offset=length * 4)
        ends.append((pool, scale))
    start = np.concatenate((np.arange(long_ones + 1) * rows, [long_ones * rows + 70])).astype(np.int32)
    lengths = np.array([length] * long_ones + [300], np.int32)
    table = np.array([0] * long_ones + [1], np.int32)
    q = raw(last.rng.standard_normal((int(start[-1]), 2 * d)), F16)
    d_start, d_lengths, d_table, d_q = (DeviceBuffer.from_numpy(x) for x in (start, lengths, table, q))
    out = DeviceBuffer(q.nbytes)
    cache = kv.KvCache(2, length, 1, d, F16, 8, ends[0][0].ptr, ends[1][0].ptr, ends[0][1].ptr, ends[1][1].ptr)
    batch = kv.KvBatch(d_start.ptr, d_lengths.ptr, d_table.ptr, long_ones + 1, 1, int(start[-1]))
    ws = kv.new_attention_workspace(cache, batch, 2, 70)
    kv.attention(cache, batch, d_q.ptr, 2, d ** -0.5, out.ptr, ws, 70)
    got = values(out.download(q.shape, np.uint16), F16)
    assert not ws.download((16384,), np.uint8).any()
    assert (np.abs(got[:long_ones * rows] - 1.0) <= 2.0 ** -11).all()       # half a step and the sum over 2^20 equal keys
    last.start = last.start + long_ones * rows
    at, want, bar, _ = rows_want(last, 2, q, 0)
    assert (np.abs(got[at].reshape(70, 2, d) - want) <= bar).all()


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("dtype,d,heads,new", [(BF16, 128, 2, 1), (F16, 64, 2, 5), (BF16, 64, 4, 3), (F16, 128, 2, 40), (BF16, 64, 2, 140)])
def test_value_scales_that_differ_between_keys(gpu, bits, dtype, d, heads, new):
    """Value scales 2^20 apart from key to key, the largest on the last tokens, which only the last rows see: every row is held relative to
    the terms it sees."""
    s = Setup([(new, 260), (new, 90 + new), (new, 141)], dtype, bits, 1, d, 16, seed=54 + new, tail=0)
    for b, (_, length) in enumerate(s.seqs):
        t = np.arange(length)
        power = np.select([t % 4 == 1, t % 7 == 3], [-20.0, 10.0], 0.0) - 5.0 * b
        if b < 2:
            power[-2:] = 12.0
        at = s.table[b, t // 16], 0, t % 16
        s.scale["v"][at] *= np.exp2(power).astype(np.float32)
    s.upload()
    q = raw(s.rng.standard_normal((s.rows, heads * d)) * 1.5, dtype)
    got = run_attention(s, heads, q, max_new=new)
    for b in range(3):
        rows, want, bar, _ = rows_want(s, heads, q, b, by_term=True)
        assert (np.abs(got[rows] - want) <= bar).all()


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("power", [118, -70])
@pytest.mark.parametrize("new", [1, 6, 50])
def test_value_scales_at_the_ends_of_bf16(gpu, bits, power, new):
    s = Setup([(new, 300), (new, new + 20)], BF16, bits, 1, 128, 16, seed=55 + new, tail=0)
    s.scale["v"] *= np.float32(2.0 ** power)
    s.upload()
    q = raw(s.rng.standard_normal((s.rows, 2 * 128)) * 1.5, BF16)
    got = run_attention(s, 2, q, max_new=new)
    for b in range(2):
        rows, want, bar, _ = rows_want(s, 2, q, b, by_term=True)
        assert (np.abs(got[rows] - want) <= bar).all()


@pytest.mark.parametrize("new,heads", [(1, 4), (30, 2)])
def test_small_probabilities_of_a_long_context_add_up(gpu, new, heads):
    """fp16: every sixteenth token takes its share of nearly all of the probability and has no value; the others have 2^-26 of such a share each."""
    length, d = 20000, 64
    s = Setup([(new, length)], F16, 16, 1, d, 64, seed=57, tail=0)
    t = np.arange(length)
    at = s.table[0, t // 64], 0, t % 64
    keys, vals = np.zeros((length, d)), s.rng.uniform(500.0, 1000.0, (length, d))
    keys[5::16, 0], vals[5::16] = 26.0 * np.log(2.0), 0.0
    s.pool["k"][at], s.pool["v"][at] = raw(keys, F16), raw(vals, F16)
    s.upload()
    q = np.zeros((new, heads, d))
    q[:, :, 0] = d ** 0.5
    q = raw(q.reshape(new, heads * d), F16)
    got = run_attention(s, heads, q, max_new=new)
    rows, want, bar, seen = rows_want(s, heads, q, 0, by_term=True)
    # a probability to 2^-32 of the largest, which is one of the shares, times the largest value
    bar = bar + (seen * 2.0 ** -32 * 1000.0 / (length / 16))[..., None]
    assert (want > 10 * bar).all() and (np.abs(got - want) <= bar).all()


@pytest.mark.parametrize("new", [1, 3, 60])
def test_sums_of_the_largest_bf16_values(gpu, new):
    s = Setup([(new, 300), (new, new + 1000)], BF16, 16, 1, 64, 16, seed=58, tail=0)
    for b, (_, length) in enumerate(s.seqs):
        t = np.arange(length)
        s.pool["v"][s.table[b, t // 16], 0, t % 16] = raw(s.rng.uniform(0.6, 0.99, (length, 64)) * 2.0 ** 128, BF16)
    s.upload()
    q = raw(s.rng.standard_normal((s.rows, 2 * 64)), BF16)
    got = run_attention(s, 2, q, max_new=new)
    for b in range(2):
        rows, want, bar, _ = rows_want(s, 2, q, b)
        assert (np.abs(got[rows] - want) <= bar).all()


@pytest.mark.parametrize("bits", [16, 8, 4])
@pytest.mark.parametrize("dtype,d,heads,kv_heads,page,window,seqs", [
    (F16, 128, 2, 1, 16, 0, [(4, 70), (3, 3), (1, 90), (2, 300)]), (BF16, 64, 4, 2, 32, 20, [(8, 200), (5, 129), (1, 40)]),
    (BF16, 128, 5, 1, 7, 0, [(3, 66), (2, 130)]), (F16, 64, 2, 2, 64, 0, [(40, 300), (9, 9), (130, 130), (1, 50)]),
    (BF16, 128, 4, 1, 16, 0, [(300, 400), (33, 200), (7, 700)]), (F16, 128, 2, 1, 24, 50, [(150, 500), (20, 140)]),
    (BF16, 64, 4, 4, 64, 90, [(130, 400)] * 40 + [(3, 60)] * 7), (F16, 128, 3, 3, 128, 0, [(200, 256), (140, 140), (11, 128)] * 20)])
def test_tokens_that_are_not_finite_reach_only_the_rows_that_see_them(gpu, bits, dtype, d, heads, kv_heads, page, window, seqs):
    """Infinities and NaN in tokens that some rows of a sequence see: the other rows have the same bits as without, and so have the other
    dimensions of the rows that see a value of them."""
    s = Setup(seqs, dtype, bits, kv_heads, d, page, seed=59, tail=0, window=window)
    q = raw(s.rng.standard_normal((s.rows, heads * d)), dtype)
    most = max(n for n, _ in seqs)
    plain = run_attention(s, heads, q, window, most)
    kept = {n: v.copy() for n, v in (s.pool if bits == 16 else s.scale).items()}
    for name in "vk":
        sees = np.zeros((s.rows, 3), bool)                # by kind: +inf, NaN, -inf (codes: +inf, NaN, +inf)
        for b, (n, length) in enumerate(seqs):
            first = length - n
            # the last token, one that half of the rows see, and with a window the first one, which only the first row sees
            tokens = [(length - 1, 0), (first + n // 2, 1)] + ([(first + 1 - window, 2)] if window and first + 1 > window else [])
            for t, kind in tokens:
                number = (np.inf, np.nan, -np.inf)[kind]
                at = s.table[b, t // page], slice(None), t % page
                if bits == 16:
                    s.pool[name][at + (5 + kind,)] = raw(np.array([number]), dtype)[0]
                else:
                    s.scale[name][at] = abs(number)
                for i in range(n):
                    if first + i >= t and (not window or first + i - t < window):
                        sees[int(s.start[b]) + i, kind] = True
        s.upload()
        got = run_attention(s, heads, q, window, most)
        any_of = sees.any(1)
        assert any_of.any() and np.array_equal(got[~any_of], plain[~any_of])
        if bits == 16 and name == "v":
            others = np.ones(d, bool)
            others[5:8] = False
            assert np.array_equal(got[:, :, others], plain[:, :, others])
            for kind in range(3):
                assert np.array_equal(got[~sees[:, kind], :, 5 + kind], plain[~sees[:, kind], :, 5 + kind])
                assert not np.isfinite(got[sees[:, kind], :, 5 + kind]).any()
        elif name == "v":
            assert not np.isfinite(got[any_of]).any()
        else:                                             # an infinite key may score -inf, which is a probability of zero
            assert np.isnan(got[sees[:, 1]]).all()
        for n, v in kept.items():
            (s.pool if bits == 16 else s.scale)[n][:] = v


def test_prefill_after_an_allocation_that_failed(gpu, monkeypatch):
    from mlxl3_b200 import decoder
    config = decoder.DecoderConfig(layers=1, hidden=256, heads=2, kv_heads=1, head_dim=128, ffn=512, vocab=512, k_bits=4, codebook=0, max_ctx=32)
    model = decoder.DenseDecoder(config, decoder.SyntheticWeights(config, seed=3))
    model.store_logits = True
    tokens = np.arange(20, dtype=np.int32)
    model.prefill(tokens[:5])
    real = decoder.new_workspace

    def out_of_memory(nbytes):
        raise gpu.B200Exl3Error("out of memory")
    monkeypatch.setattr(decoder, "new_workspace", out_of_memory)
    with pytest.raises(gpu.B200Exl3Error, match="out of memory"):
        model.prefill(tokens)
    model.prefill(tokens[:5])                            # what was there still is
    monkeypatch.setattr(decoder, "new_workspace", real)
    model.prefill(tokens)
    fresh = decoder.DenseDecoder(config, decoder.SyntheticWeights(config, seed=3))
    fresh.store_logits = True
    fresh.prefill(tokens)
    assert np.array_equal(model.download("logits"), fresh.download("logits"))


def test_lengths_and_rows_without_sense(gpu):
    """The largest and smallest lengths, first rows before the buffers: the largest length counts as 2^30 tokens, of which the table's are seen;
    rows of no sequence, of tokens before the first, and all pages stay as they are."""
    heads, d = 4, 64
    s = Setup([(5, 48), (4, 40), (3, 30)], F16, 16, 2, d, 16, seed=61, gap=2)
    for length, first in (((1 << 31) - 1, 2), (1 << 30, 2), ((1 << 31) - 1, -(1 << 31))):
        s.d_start.upload(np.array([first, 7, 11, 14], np.int64).astype(np.int32))
        s.d_length.upload(np.array([length, -(1 << 31), 30], np.int64).astype(np.int32))
        n0 = 7 - max(first, 0)
        width = (heads + 4) * d
        qkv = raw(s.rng.standard_normal((s.rows, width)), F16)
        turns = s.kv.rope_turns(d, 10000.0)
        d_qkv, d_turns = s.Buffer.from_numpy(qkv), s.Buffer.from_numpy(turns)
        sentinel = raw(np.full((s.rows, heads * d), 9.0), F16)
        out, read = s.Buffer.from_numpy(sentinel), s.Buffer.from_numpy(np.full((s.rows, 2, d), 5.0, np.float32))
        batch = s.kv.KvBatch(s.d_start.ptr, s.d_length.ptr, s.d_table.ptr, 2, s.width, s.rows)           # the third sequence only reads
        s.kv.append(s.cache, batch, d_qkv.ptr + heads * d * 2, d_qkv.ptr + (heads + 2) * d * 2, s.kv.Rope(d_turns.ptr, d), d_qkv.ptr, heads, d_qkv.ptr,
                    width, width, width, width)
        ws = s.kv.new_attention_workspace(s.cache, batch, heads)
        s.kv.attention(s.cache, batch, d_qkv.ptr, heads, d ** -0.5, out.ptr, ws, q_stride=width)
        s.kv.read(s.cache, s.batch, F32, read.ptr, 0)
        pool, _ = s.download()
        assert all(np.array_equal(pool[n], s.pool[n]) for n in "kv")                  # nothing lay in the table
        rotated, got = d_qkv.download(qkv.shape, np.uint16), out.download(sentinel.shape, np.uint16)
        ours = np.arange(s.rows)
        ours = (ours >= max(first, 0)) & (ours < 7)
        assert np.array_equal(rotated[~ours], qkv[~ours]) and np.array_equal(rotated[:, heads * d:], qkv[:, heads * d:])
        keys, vals = np.zeros((64, 2, d)), np.zeros((64, 2, d))                       # the table's last page is none: zeros
        keys[:48], vals[:48] = s.held("k", 0, np.arange(48)), s.held("v", 0, np.arange(48))
        position = (1 << 30) - n0
        for i, row in enumerate(np.flatnonzero(ours)):
            q = values(rotated[row, :heads * d], F16).reshape(heads, d)
            x = values(qkv[row, :heads * d], F16).reshape(heads, d)
            # turns in 64 bits at 2^30 are off by 2^30 * 2^-53 of a turn; then fp32 and one rounding to fp16
            assert np.abs(q - okv.rope(x, position + i, turns)).max() <= (2.0 ** -11 + 2.0 ** -19) * 8
            want, mass, most, seen, top_v = okv.attention(q[None], keys, vals, position + i, d ** -0.5)
            bar = (np.expm1(2 * (d + 4) * 2.0 ** -23 * most) + 2.0 ** -20 + 2.0 ** -11 + seen * 2.0 ** -22)[..., None] * mass + (2.0 ** -25 * seen * top_v)[..., None]
            bar = bar + 2.0 ** -11 * (np.abs(want) + bar) + 2.0 ** -25
            assert (seen == 64).all() and (np.abs(values(got[row], F16).reshape(1, heads, d) - want) <= bar).all()
        assert (got[7:11] == 0).all()                                                 # a sequence without tokens
        none = ~ours
        none[7:11] = False
        assert np.array_equal(got[none], sentinel[none])
        back = read.download((s.rows, 2, d), np.float32)
        assert np.array_equal(back[11:14], s.held("k", 2, np.array([27, 28, 29])).astype(np.float32)) and (np.delete(back, [11, 12, 13], 0) == 5.0).all()
        assert not ws.download((16384,), np.uint8).any()


@pytest.mark.parametrize("bits", [16, 8, 4])
def test_single_tokens_beside_one_that_is_not_finite(gpu, bits):
    """A step of single tokens: a sequence that holds an infinity and one that holds a NaN are not finite, the others have the same bits."""
    s = Setup([(1, 90), (1, 200), (1, 17), (1, 300)], BF16, bits, 2, 128, 16, seed=62, tail=0)
    q = raw(s.rng.standard_normal((s.rows, 4 * 128)), BF16)
    plain = run_attention(s, 4, q, max_new=1)
    for b, t, number in ((1, 199, np.inf), (2, 3, np.nan)):
        at = s.table[b, t // 16], slice(None), t % 16
        if bits == 16:
            s.pool["v"][at + (9,)] = raw(np.array([number]), BF16)[0]
        else:
            s.scale["v"][at] = number
    s.upload()
    got = run_attention(s, 4, q, max_new=1)
    assert np.array_equal(got[[0, 3]], plain[[0, 3]])
    odd = np.ones(128, bool)
    if bits == 16:
        odd[:] = False
        odd[9] = True
        assert np.array_equal(got[1:3][:, :, ~odd], plain[1:3][:, :, ~odd])
    assert not np.isfinite(got[1:3][:, :, odd]).any()
